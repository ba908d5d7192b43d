"""The cases by which the dense-layer operators (kaldi_amd/dense.py) are measured.

Three operators of a residual acoustic network, served frame by frame or over whole batches:

  norm     s = x + r;  y = s / sqrt(mean(s^2) + eps) * w        (x, r: one type; s is returned too)
  convert  y = x in another type                                 (the way into 16 and 8 bits)
  linear   y = act(x W^T + b) + r                                (16- or 8-bit x and W)

8 bits ("mx8") means e4m3 values with one power-of-two scale (e8m0) per 32 consecutive columns of
a row: the smallest power of two 2^k, k >= -127, with max|group| <= 448 * 2^k.

`own = False`: plain torch operations in 32 bits, rounded once at the end.  `own = True`: the calls
of kaldi_amd.dense.  An mx8 output is returned as its e4m3 values and its scales, both in the
8-bit floating types that stand for them.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4.0, "bf16": 2.0, "f16": 2.0, "mx8": 1.0 + 1.0 / 32}
ACTS = ("none", "relu", "sigmoid", "tanh", "silu", "gelu")


def listed():
    def norm(name, rows, dim, type_, out, residual, weight, pad=0):
        return {"name": name, "op": "norm", "rows": rows, "dim": dim, "type": type_, "out": out,
                "residual": residual, "weight": weight, "pad": pad}

    def convert(name, rows, dim, type_, out, pad=0):
        return {"name": name, "op": "convert", "rows": rows, "dim": dim, "type": type_, "out": out, "pad": pad}

    def linear(name, rows, k, n, type_, out, act, residual, pad=0):
        return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "type": type_, "out": out,
                "act": act, "residual": residual, "pad": pad}

    return [
        # one frame of one stream on its way into an 8-bit layer
        norm("norm one frame", 1, 2048, "bf16", "mx8", True, True),
        # the p-norm net's normalised layer (200 wide) over bench's launch of 35 554 frames
        norm("norm narrow f32", 35554, 200, "f32", "bf16", False, False),
        # an odd width without padding between the rows: no row but the first starts on 16 bytes
        norm("norm odd f16", 1237, 1999, "f16", "f16", True, True),
        # a batch of frames of a wide residual network, into an 8-bit layer
        norm("norm batch", 16384, 4096, "bf16", "mx8", True, True),
        # one chunk of spliced features (9 x 40) of an online decoder, into 8 bits
        convert("convert chunk", 64, 360, "f32", "mx8"),
        # activations of the net's hidden width over the launch of 35 554 frames
        convert("convert batch", 35554, 2000, "bf16", "mx8"),
        # one frame through one layer: latency
        linear("linear one frame", 1, 2048, 2048, "bf16", "bf16", "silu", False),
        # 16 streams decoded side by side, 8 bits, back onto the residual stream
        linear("linear 16 streams", 16, 4096, 4096, "mx8", "bf16", "none", True),
        # one utterance of 3 s through the net's first hidden layer (360 -> 2000)
        linear("linear utterance", 300, 360, 2000, "f16", "f16", "relu", False),
        # odd sizes, rows that start anywhere
        linear("linear odd", 1237, 1999, 2001, "bf16", "f32", "tanh", True),
        # hidden width to the 8 600 pdfs' logits over the launch of 35 554 frames
        linear("linear logits", 35554, 2000, 8600, "bf16", "f32", "none", False),
        # the wide half of a feed-forward pair over a batch, 8 bits in and out
        linear("linear wide mx8", 8192, 4096, 16384, "mx8", "mx8", "gelu", False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "convert", "linear", "linear", "linear"])
    rows = _log_int(rng, 1, 36000)
    if op != "linear":
        dim = min(_log_int(rng, 48, 12000), (1 << 26) // rows)
        case = {"op": op, "rows": rows, "dim": dim, "type": rng.choice(["f32", "bf16", "f16"]),
                "pad": rng.choice([0, 0, 8, 5])}
        case["out"] = rng.choice(["mx8", "mx8"] + [t for t in TYPES if op == "norm" or t != case["type"]])
        if op == "norm":
            case.update(residual=rng.random() < 0.7, weight=rng.random() < 0.7)
        return case
    type_ = rng.choice(["bf16", "f16", "mx8"])
    k, n = _log_int(rng, 64, 8192), _log_int(rng, 64, 16384)
    if rng.random() < 0.6:  # widths of real layers: mostly multiples of 8
        k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
    rows = max(1, min(rows, int(1.0e12 / (2.0 * k * n)), (1 << 28) // n))
    return {"op": "linear", "rows": rows, "k": k, "n": n, "type": type_,
            "out": rng.choice(["mx8", "f32"] + [type_ if type_ != "mx8" else "bf16"] * 2),
            "act": rng.choice(ACTS), "residual": rng.random() < 0.5, "pad": rng.choice([0, 0, 8, 5])}


def work(case):
    rows = case["rows"]
    if case["op"] != "linear":
        dim, b = case["dim"], BYTES[case["type"]]
        per = b + BYTES[case["out"]]
        if case["op"] == "norm" and case["residual"]:
            per += 2 * b  # the residual in, the sum out
        weight = 4.0 * dim if case.get("weight") else 0.0
        return {"bytes": rows * dim * per + weight, "flops": 4.0 * rows * dim}
    k, n, b = case["k"], case["n"], BYTES[case["type"]]
    total = rows * k * b + n * k * b + 4.0 * n + rows * n * BYTES[case["out"]]
    if case["residual"]:
        total += rows * n * BYTES[_residual_type(case)]
    return {"bytes": total, "flops": 2.0 * rows * k * n}


def _residual_type(case):
    return case["out"] if case["out"] != "mx8" else "bf16"


# ---- mx8 in plain torch -------------------------------------------------------------------------

def _groups(t):
    rows, dim = t.shape
    return torch.nn.functional.pad(t, (0, -dim % 32)).view(rows, -1, 32)


def _to_mx8(y):
    """float values -> (e4m3 values, e8m0 scales); what is not finite becomes NaN."""
    dim = y.shape[1]
    g = _groups(y)
    finite = torch.isfinite(g)
    amax = torch.where(finite, g.abs(), torch.zeros_like(g)).amax(2)
    m, e = torch.frexp(amax)
    k = torch.where(amax > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, -127)).clamp(-127, 127)
    half = k // 2  # 2^-k in two factors: neither leaves the range of 32 bits
    one = torch.ones_like(amax)
    q = g * torch.ldexp(one, -half).unsqueeze(2) * torch.ldexp(one, half - k).unsqueeze(2)
    q = torch.where(finite, q, torch.full_like(q, math.nan))
    q = q.reshape(y.shape[0], -1)[:, :dim].to(torch.float8_e4m3fn).contiguous()
    return q, (k + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _from_mx8(q, scales, type_=torch.float32):
    rows, dim = q.shape
    return (_groups(q.to(type_)) * scales.to(type_).unsqueeze(2)).view(rows, -1)[:, :dim]


def _result(y, out):
    if out == "mx8":
        q, scales = _to_mx8(y)
        return {"values": q, "scales": scales}
    return {"y": y.to(TYPES[out])}


# ---- inputs ---------------------------------------------------------------------------------------

def _padded(rows, cols, pad, dtype):
    """A [rows x cols] view of a buffer with `pad` more columns."""
    return torch.zeros((rows, cols + pad), dtype=dtype, device="cuda")[:, :cols]


def _frames(rows, dim, g, loud):
    """Activations as a residual stream carries them: rows of different loudness, and a few columns
    that are much larger than the rest."""
    x = torch.randn((rows, dim), generator=g, device="cuda")
    if loud:
        x *= torch.exp(0.7 * torch.randn((rows, 1), generator=g, device="cuda"))
        x *= 1 + 20 * (torch.rand((1, dim), generator=g, device="cuda") < 0.01)
    return x


def _out_buffers(case, rows, n):
    out = case["out"]
    if out == "mx8":
        ld = (n + 31) // 32 * 32
        return {"values": torch.zeros((rows, ld), dtype=torch.float8_e4m3fn, device="cuda")[:, :n],
                "scales": torch.zeros((rows, ld // 32), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)}
    return {"y": _padded(rows, n, case["pad"], TYPES[out])}


def _matrix(dense, t, type_, scales=None):
    return dense.Matrix(t.data_ptr(), type_, t.stride(0), scales.data_ptr() if scales is not None else 0,
                        scales.stride(0) if scales is not None else 0)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    rows, pad = case["rows"], case["pad"]
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        w = torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k)
        x = _frames(rows, k, g, False)
        if case["type"] == "mx8":
            s["w"], s["w_scales"] = _to_mx8(w)
            w = _from_mx8(s["w"], s["w_scales"])
            q, s["x_scales"] = _to_mx8(x)
            s["x"] = _padded(rows, k, -k % 16 if pad != 5 else pad, torch.uint8).view(torch.float8_e4m3fn)
            s["x"].copy_(q)
        else:
            s["w"] = w.to(TYPES[case["type"]])
            w = s["w"].float()
            s["x"] = _padded(rows, k, pad, TYPES[case["type"]])
            s["x"].copy_(x)
        s["b"] = 0.1 * torch.randn((n,), generator=g, device="cuda")
        if case["residual"]:
            s["r"] = _padded(rows, n, pad, TYPES[_residual_type(case)])
            s["r"].copy_(_frames(rows, n, g, False))
        if own:
            from kaldi_amd import dense
            s["handle"] = dense.Linear(w.cpu().numpy(), s["b"].cpu().numpy(), case["type"])
            s["out"] = _out_buffers(case, rows, n)
            s["mx"] = _matrix(dense, s["x"], case["type"], s.get("x_scales"))
            s["mr"] = _matrix(dense, s["r"], _residual_type(case)) if case["residual"] else None
    else:
        dim = case["dim"]
        s["x"] = _padded(rows, dim, pad, TYPES[case["type"]])
        s["x"].copy_(_frames(rows, dim, g, True))
        if case["op"] == "norm":
            if case["residual"]:
                s["r"] = _padded(rows, dim, pad, TYPES[case["type"]])
                s["r"].copy_(_frames(rows, dim, g, True))
            if case["weight"]:
                s["w"] = 1 + 0.2 * torch.randn((dim,), generator=g, device="cuda")
        if own:
            from kaldi_amd import dense
            s["out"] = _out_buffers(case, rows, dim)
            s["mx"] = _matrix(dense, s["x"], case["type"])
            s["mr"] = s["ms"] = None
            if case["op"] == "norm":
                s["handle"] = dense.RmsNorm(dim, s["w"].cpu().numpy() if case["weight"] else None, EPS)
                if case["residual"]:
                    s["mr"] = _matrix(dense, s["r"], case["type"])
                    s["out"]["sum"] = _padded(rows, dim, pad, TYPES[case["type"]])
                    s["ms"] = _matrix(dense, s["out"]["sum"], case["type"])
    if own:
        from kaldi_amd import dense
        o = s["out"]
        s["mo"] = _matrix(dense, o["values"], "mx8", o["scales"]) if case["out"] == "mx8" else _matrix(dense, o["y"], case["out"])
    return s


# ---- one pass -------------------------------------------------------------------------------------

def _run_own(s):
    from kaldi_amd import dense
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "norm":
        s["handle"].ApplyDevice(s["mx"], case["rows"], s["mo"], residual=s["mr"], sum=s["ms"], stream=stream)
    elif case["op"] == "convert":
        dense.ConvertDevice(s["mx"], case["rows"], case["dim"], s["mo"], stream=stream)
    else:
        s["handle"].ApplyDevice(s["mx"], case["rows"], s["mo"], activation=case["act"], residual=s["mr"], stream=stream)
    return s["out"]


def _activate(y, act):
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-y))
    if act == "tanh":
        return torch.tanh(y)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["op"] == "convert":
        return _result(s["x"].float(), case["out"])
    if case["op"] == "norm":
        h = s["x"].float()
        if case["residual"]:
            h = h + s["r"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
        if case["weight"]:
            y = y * s["w"]
        out = _result(y, case["out"])
        if case["residual"]:
            out["sum"] = h.to(TYPES[case["type"]])
        return out
    if case["type"] == "mx8":
        x, w = _from_mx8(s["x"], s["x_scales"]), _from_mx8(s["w"], s["w_scales"])
    else:
        x, w = s["x"].float(), s["w"].float()
    y = _activate(torch.matmul(x, w.t()) + s["b"], case["act"])
    if case["residual"]:
        y = y + s["r"].float()
    return _result(y, case["out"])


# ---- the definition in 64 bits ----------------------------------------------------------------------

def _exact_result(y, out):
    """An mx8 output is given before its values' rounding, in units of the group's scale.  The scale
    itself has no value here: where a group's largest number lies within a rounding of a border, two
    neighbouring powers of two are equally right."""
    if out != "mx8":
        return {"y": y}
    rows, dim = y.shape
    top = torch.nn.functional.pad(y.abs(), (0, -dim % 32)).view(rows, -1, 32).max(dim=2).values
    k = torch.ceil(torch.log2(top / 448)).clamp(min=-127)
    return {"values": y * torch.exp2(-k).repeat_interleave(32, dim=1)[:, :dim], "scales": None}


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "convert":
        return _exact_result(x, case["out"])
    if case["op"] == "norm":
        total = x + s["r"].double() if case["residual"] else x
        length = torch.linalg.vector_norm(total, dim=1, keepdim=True)
        y = total / torch.sqrt(length ** 2 / case["dim"] + EPS)
        out = _exact_result(y * s["w"].double() if case["weight"] else y, case["out"])
        if case["residual"]:
            out["sum"] = total
        return out
    w = s["w"].double()
    if case["type"] == "mx8":
        x = x * s["x_scales"].double().repeat_interleave(32, dim=1)[:, :case["k"]]
        w = w * s["w_scales"].double().repeat_interleave(32, dim=1)[:, :case["k"]]
    y = torch.addmm(s["b"].double(), x, w.t())
    act = {"none": lambda v: v, "relu": torch.relu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
           "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[case["act"]]
    y = act(y)
    if case["residual"]:
        y = y + s["r"].double()
    return _exact_result(y, case["out"])
