"""Sizes that take each form of the linear kernels on 256 compute units, and what says which."""
import re

from kaldi_amd import dense

UNITS = 256

# (layer's type, output's type, rows, k, n, whether rows of x start and end on 16 bytes)
CASES = [
    ("bf16", "f32", 200, 520, 130, True), ("f16", "f32", 200, 520, 130, True), ("bf16", "mx8", 7, 513, 333, False),
    ("f16", "mx8", 7, 513, 333, False), ("bf16", "mx8", 9, 520, 333, True), ("f16", "mx8", 9, 520, 333, True),
    ("bf16", "bf16", 300, 96, 264, True), ("f16", "f16", 300, 96, 264, True), ("bf16", "f32", 257, 520, 513, True),
    ("f16", "f32", 257, 520, 513, True), ("bf16", "f32", 640, 136, 520, True), ("f16", "f32", 640, 136, 520, True),
    ("mx8", "bf16", 20, 1168, 130, True), ("mx8", "f32", 20, 1168, 130, True), ("mx8", "mx8", 20, 1071, 130, False),
    ("mx8", "bf16", 300, 96, 264, True), ("mx8", "f32", 300, 96, 264, True), ("mx8", "f32", 300, 97, 264, False),
    ("mx8", "f32", 17, 2000, 4400, True), ("mx8", "f32", 9, 1999, 5100, False), ("mx8", "bf16", 200, 1984, 1032, True),
    ("mx8", "f32", 257, 520, 513, False),
    # 64 x 32 in 8 bits (two k-tiles of a wave at once): odd numbers of k-tiles, last groups that are short
    ("mx8", "bf16", 977, 1211, 409, False), ("mx8", "mx8", 977, 1211, 409, False), ("mx8", "f32", 468, 2281, 975, False),
    ("mx8", "f32", 256, 4096, 2048, True), ("mx8", "f32", 250, 4112, 2000, True), ("mx8", "bf16", 930, 1168, 409, True),
    ("mx8", "mx8", 930, 656, 409, True),
    # tiles of 64 x 64, copied: one block for each, several; two groups of waves
    ("bf16", "f32", 990, 200, 2000, True), ("f16", "f16", 990, 200, 2000, True), ("bf16", "bf16", 60000, 200, 60, True),
    ("f16", "f32", 60000, 200, 60, True), ("mx8", "bf16", 990, 400, 2000, True), ("mx8", "f32", 990, 400, 2000, True),
    ("mx8", "bf16", 60000, 400, 60, True), ("mx8", "f32", 60000, 400, 60, True), ("bf16", "f32", 500, 1000, 2000, True),
    ("f16", "bf16", 500, 1000, 2000, True), ("mx8", "bf16", 500, 2000, 2000, True), ("mx8", "f32", 500, 2000, 2000, True),
    # through registers: one block for each, several
    ("bf16", "f32", 500, 1017, 2000, False), ("f16", "f32", 500, 1017, 2000, False), ("mx8", "bf16", 500, 2017, 2000, False),
    ("mx8", "f32", 640, 139, 520, False), ("bf16", "f32", 1198, 1412, 13286, False), ("f16", "bf16", 34900, 331, 130, False),
    ("mx8", "mx8", 76643, 1327, 27, False), ("mx8", "f32", 76643, 1327, 27, False), ("mx8", "bf16", 68800, 331, 17, False),
    # tiles of 128 x 128, copied, in one and two groups, and through registers
    ("bf16", "bf16", 3990, 200, 1990, True), ("f16", "f32", 3990, 200, 1990, True), ("bf16", "f32", 4090, 200, 4600, True),
    ("f16", "f16", 4090, 200, 4600, True), ("mx8", "bf16", 3990, 400, 1990, True), ("mx8", "f32", 3990, 400, 1990, True),
    ("mx8", "bf16", 4090, 400, 4600, True), ("mx8", "f32", 4090, 400, 4600, True), ("bf16", "f32", 1990, 1000, 1990, True),
    ("f16", "f32", 1990, 1000, 1990, True), ("bf16", "f32", 90000, 504, 120, True), ("f16", "bf16", 90000, 504, 120, True),
    ("mx8", "bf16", 1990, 2000, 1990, True), ("mx8", "f32", 1990, 2000, 1990, True), ("mx8", "bf16", 90000, 1008, 120, True),
    ("mx8", "f32", 90000, 1008, 120, True), ("bf16", "f32", 9000, 65, 520, False), ("f16", "f32", 9000, 65, 520, False),
    ("bf16", "mx8", 44730, 331, 129, False), ("f16", "f32", 44730, 331, 129, False), ("mx8", "bf16", 9000, 65, 520, False),
    ("mx8", "f32", 9000, 65, 520, False), ("mx8", "mx8", 44730, 331, 129, False), ("mx8", "f32", 44730, 331, 129, False),
    # tiles of 256 x 256
    ("bf16", "f32", 4090, 1000, 4090, True), ("f16", "bf16", 4090, 1000, 4090, True), ("bf16", "bf16", 8000, 200, 8000, True),
    ("f16", "f32", 8000, 200, 8000, True), ("mx8", "bf16", 4090, 2000, 4090, True), ("mx8", "bf16", 8000, 400, 8000, True),
]


def form(type_, out, rows, k, n, aligned):
    """(kernel and its arguments, whether a block has several tiles)."""
    text = dense.linear_kernel_info(type_, out, rows, k, n, aligned, UNITS)
    counts = re.search(r"tiles=(\d+) blocks=(\d+)", text)
    return text.split()[0], bool(counts) and int(counts[1]) > int(counts[2])


def is_aligned(type_, k, ld, ld_scales):
    """Of a matrix whose first row starts on 16 bytes."""
    es = 1 if type_ == "mx8" else 2
    return k * es % 16 == 0 and ld * es % 16 == 0 and (type_ != "mx8" or ld_scales % 16 == 0)
