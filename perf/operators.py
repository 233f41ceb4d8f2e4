"""Cases and plain forms of the quantised linear layer's operators.

A linear layer trained or served from what the update step emits: products
with the 4-bit weights as they lie (forward and input gradient), activations
kept in 8 bits between the two passes, and the weight gradient taken from
them.  Each case names one operator:

    linear  y[m, n]  = sum_k x[m, k] W[n, k]      W in 4 bits with block scales
    dgrad   dx[m, k] = sum_n dy[m, n] W[n, k]
    act8    x -> 8-bit codes with a power of two per 32 columns -> x'
    wgrad   dW[n, k] = alpha sum_m dy[m, n] x'[m, k] (+ add[n, k])

W's bytes are the framework's: blocks over the flattened [out, in] weight,
MXFP4 32 elements in 17 bytes (16 of codes, element 2i in the high nibble,
then the E8M0 scale), NVFP4 16 elements in 9 bytes (8 of codes, then the
E4M3 scale).  A block may straddle two rows.
"""
import math

import numpy as np
import torch

own = False

if own:
    import odyssey_b200  # noqa: F401

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NAMES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
# 4-bit kinds: elements per block, bytes per block, library kind code
KINDS = {"mxfp4": (32, 17, 6), "nvfp4": (16, 9, 7), "nvfp4_tensor": (16, 9, 8), "mxfp4_ocp": (32, 17, 9)}
# 8-bit formats: mantissa bits, smallest normal exponent, largest value, the exponent of its power of two, scale range
FORMATS = {"e4m3": (3, -6, 448.0, 8, -117, 119), "e5m2": (2, -14, 57344.0, 15, -110, 112)}
LARGEST = 8192 * 4096 * 4096


def listed():
    return [
        # the last layer of a small classifier (LeNet's 120 x 400), a batch of 32: launches and host calls only
        {"name": "linear lenet fc f32", "op": "linear", "kind": "mxfp4", "rows": 32, "out": 120, "in": 400, "dtype": "f32",
         "strided": False},
        # one new token in serving, the 4096 x 4096 layer of the flat model, weights as its step leaves them
        {"name": "linear token 4096", "op": "linear", "kind": "nvfp4_tensor", "rows": 1, "out": 4096, "in": 4096,
         "dtype": "bf16", "strided": False},
        # one token for each of 8 users, a wide layer: the weights' bytes from memory
        {"name": "linear 8 tokens 8192", "op": "linear", "kind": "mxfp4", "rows": 8, "out": 8192, "in": 8192, "dtype": "bf16",
         "strided": False},
        # a short ragged batch, rows whose blocks straddle, taken out of a wider buffer
        {"name": "linear ragged f16", "op": "linear", "kind": "mxfp4_ocp", "rows": 37, "out": 1000, "in": 2056, "dtype": "f16",
         "strided": True},
        # a prompt or a training batch through the flat model's layer
        {"name": "linear prompt 2048", "op": "linear", "kind": "nvfp4", "rows": 2048, "out": 4096, "in": 4096, "dtype": "bf16",
         "strided": False},
        # the input gradient of a training step on the flat model's layer
        {"name": "dgrad 4096 tokens", "op": "dgrad", "kind": "nvfp4_tensor", "rows": 4096, "out": 4096, "in": 4096,
         "dtype": "bf16", "strided": False},
        # the input gradient of a handful of positions (fine-tuning on the last tokens), float32 gradients
        {"name": "dgrad 4 rows f32", "op": "dgrad", "kind": "mxfp4", "rows": 4, "out": 4096, "in": 4096, "dtype": "f32",
         "strided": False},
        # one layer's input kept for the backward pass and brought back
        {"name": "act8 e4m3 bf16", "op": "act8", "format": "e4m3", "rows": 8192, "in": 4096, "dtype": "bf16", "strided": False},
        # a ragged float32 activation with a wide range
        {"name": "act8 e5m2 f32 ragged", "op": "act8", "format": "e5m2", "rows": 1021, "in": 1037, "dtype": "f32",
         "strided": False},
        # the weight gradient of a full training batch, in the step's gradient type
        {"name": "wgrad 8192 tokens", "op": "wgrad", "format": "e4m3", "rows": 8192, "out": 4096, "in": 4096, "dtype": "bf16",
         "grad": "bf16", "add": False},
        # a convolution's weight as a matrix (512 x 4608), float16 gradients, accumulated over micro-batches in float32
        {"name": "wgrad 512x4608 f16 add", "op": "wgrad", "format": "e5m2", "rows": 2048, "out": 512, "in": 4608, "dtype": "f16",
         "grad": "f32", "add": True},
        # a small ragged layer in float32
        {"name": "wgrad ragged f32", "op": "wgrad", "format": "e4m3", "rows": 333, "out": 1000, "in": 515, "dtype": "f32",
         "grad": "f32", "add": False},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "dgrad", "act8", "wgrad"))
    while True:
        rows = _log_uniform(rng, 1, 8192)
        n, k = _log_uniform(rng, 8, 8192), _log_uniform(rng, 8, 8192)
        if rng.random() < 0.6:  # most layers have widths of whole tiles
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        elif rng.random() < 0.5:
            n, k = n | 1, k | 1
        if rows * n * k <= LARGEST:
            break
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op in ("linear", "dgrad"):
        return {"op": op, "kind": rng.choice(sorted(KINDS)), "rows": rows, "out": n, "in": k, "dtype": dtype,
                "strided": rng.random() < 0.25}
    if op == "act8":
        return {"op": op, "format": rng.choice(sorted(FORMATS)), "rows": rows, "in": k, "dtype": dtype,
                "strided": rng.random() < 0.25}
    return {"op": op, "format": rng.choice(sorted(FORMATS)), "rows": rows, "out": n, "in": k, "dtype": dtype,
            "grad": rng.choice(("f32", "bf16", dtype)), "add": rng.random() < 0.3}


def _quant_bytes(kind, n):
    block, size, _ = KINDS[kind]
    return -(-n // block) * size


def work(case):
    rows, k, e = case["rows"], case["in"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "act8":
        kept = rows * (-(-k // 32)) * 33
        return {"bytes": 2 * (rows * k * e + kept), "flops": 4 * rows * k}
    n = case["out"]
    flops = 2 * rows * n * k
    if case["op"] == "wgrad":
        g = DTYPES[case["grad"]].itemsize
        return {"bytes": rows * n * e + rows * (-(-k // 32)) * 33 + n * k * g * (2 if case["add"] else 1), "flops": flops}
    return {"bytes": _quant_bytes(case["kind"], n * k) + rows * (n + k) * e, "flops": flops}


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=gen.device, dtype=torch.float32)


def _rows(gen, rows, cols, dtype, strided, scale=1.0, spread=0.0):
    """Rows of activations or gradients: N(0, scale^2), with `spread` a range that differs from row to row and a few
    outliers, as activations have; `strided`: columns of a wider buffer."""
    x = _normal(gen, rows, cols) * scale
    if spread:
        x = x * torch.exp2(_normal(gen, rows, 1) * spread)
        x = torch.where(torch.rand(rows, cols, generator=gen, device=gen.device) < 1e-3, x * 50.0, x)
    x = x.to(dtype)
    if not strided:
        return x
    wide = torch.zeros(rows, cols + 24, device=gen.device, dtype=dtype)
    wide[:, 8:8 + cols] = x
    return wide[:, 8:8 + cols]


def _weights(gen, kind, n, k):
    """A weight's bytes: N(0, 0.02^2) quantised block by block."""
    block, size, _ = KINDS[kind]
    numel = n * k
    blocks = -(-numel // block)
    w = torch.zeros(blocks * block, device=gen.device)
    w[:numel] = _normal(gen, numel) * 0.02
    ts = 1.0
    if kind == "nvfp4_tensor":
        ts = float(np.float32(float(w.abs().max()) / 2688.0))
        w = w / ts
    w = w.view(blocks, block)
    amax = w.abs().amax(1)
    if size == 17:
        e = torch.frexp(amax).exponent.to(torch.int32) - 3
        e = e.clamp(-126, 126)
        scale_byte, scale = (e + 127).to(torch.uint8), _pow2(e)
    else:
        scale = (amax / 6.0).clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn)
        scale_byte, scale = scale.view(torch.uint8), scale.float()
    q = w / scale[:, None]
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=gen.device)
    mag = torch.bucketize(q.abs(), edges)
    if kind != "mxfp4_ocp":
        mag = torch.where(mag == 1, 2, mag)
    code = (mag + 8 * (q < 0)).to(torch.uint8)
    packed = torch.empty(blocks, size, dtype=torch.uint8, device=gen.device)
    packed[:, :size - 1] = code[:, 0::2] * 16 + code[:, 1::2]
    packed[:, size - 1] = scale_byte
    return packed.view(-1), ts


def _groups(x):
    """x [rows, cols] as float32 groups of 32 columns, the last filled up with zeros."""
    rows, cols = x.shape
    g = -(-cols // 32)
    p = torch.zeros(rows, g * 32, device=x.device)
    p[:, :cols] = x
    return p.view(rows, g, 32)


def _encode8(x, fmt):
    """Values (as multiples of the scale) and exponents of the 8-bit form, by the definition: the least power of two
    with amax <= largest * 2^X, values rounded to the format's grid, ties to even."""
    mant, emin, largest, top, xmin, xmax = FORMATS[fmt]
    p = _groups(x)
    m, e = torch.frexp(p.abs().amax(2))
    power = torch.where(m <= 0.875, e - 1 - top, e - top).clamp(xmin, xmax)
    power = torch.where(m == 0, xmin, power)
    v = p * _pow2(-power[:, :, None])
    step = _pow2((torch.frexp(v).exponent - 1).clamp(min=emin) - mant)
    v = (torch.round(v / step) * step).clamp(-largest, largest)
    return v, power


def _codes8(v, fmt):
    """The bytes that stand for values on the format's grid."""
    mant, emin, _, _, _, _ = FORMATS[fmt]
    m, e = torch.frexp(v.abs())
    e = e - 1
    bias = 1 - emin
    normal = ((e + bias) * 2 ** mant).float() + (m * 2 - 1) * 2 ** mant
    subnormal = v.abs() * 2.0 ** (mant - emin)
    code = torch.where(v.abs() >= 2.0 ** emin, normal, subnormal).to(torch.int32)
    return (code + 128 * torch.signbit(v)).to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    dtype, rows, k, op = DTYPES[case["dtype"]], case["rows"], case["in"], case["op"]
    s = dict(case)
    if op == "linear":
        s["x"] = _rows(gen, rows, k, dtype, case["strided"], spread=0.5)
        s["q"], s["scale"] = _weights(gen, case["kind"], case["out"], k)
    elif op == "dgrad":
        s["x"] = _rows(gen, rows, case["out"], dtype, case["strided"], scale=0.1)
        s["q"], s["scale"] = _weights(gen, case["kind"], case["out"], k)
    elif op == "act8":
        s["x"] = _rows(gen, rows, k, dtype, case["strided"], spread=2.0)
    else:
        s["dy"] = _rows(gen, rows, case["out"], dtype, False, scale=0.1)
        v, power = _encode8(_rows(gen, rows, k, torch.float32, False, spread=0.5), case["format"])
        s["codes"] = _codes8(v, case["format"]).view(rows, -1)
        s["scales"] = (power + 127).to(torch.uint8)
        if case["add"]:
            s["sum"] = _normal(gen, case["out"], k).to(DTYPES[case["grad"]])
    return s


def _pow2(e):
    """2^e in float32 for whole e from -126 to 127, exactly (the exponent's bits)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _pow2_64(e):
    """2^e in float64 for whole e from -200 to 200, exactly (looked up)."""
    return torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=e.device)[e.long() + 200]


def _e2m1(kind, device):
    half = 0.5 if kind == "mxfp4_ocp" else 0.0
    t = [0.0, half, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(t + [-v for v in t], device=device)


def _plain_weight(s):
    """W [out, in] in float32, without the tensor scale."""
    block, size, _ = KINDS[s["kind"]]
    b = s["q"].view(-1, size)
    code = torch.stack((b[:, :-1] >> 4, b[:, :-1] & 15), 2).view(-1, block).int()
    byte = b[:, -1:].int()
    if size == 17:
        scale = _pow2(byte - 127)
    else:
        e, m = (byte >> 3) & 15, (byte & 7).float()
        scale = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * _pow2(e - 7))
    w = _e2m1(s["kind"], b.device)[code] * scale
    return w.reshape(-1)[:s["out"] * s["in"]].view(s["out"], s["in"])


def _plain_values8(codes, scales, cols, fmt):
    mant, emin, _, _, _, _ = FORMATS[fmt]
    c = codes.int()
    e, m = (c & 127) >> mant, (c & (2 ** mant - 1)).float() / 2 ** mant
    v = torch.where(e == 0, m * 2.0 ** emin, (1 + m) * _pow2(e + emin - 1))
    v = torch.where(c >= 128, -v, v) * _pow2(scales.int() - 127).repeat_interleave(32, 1)
    return v[:, :cols]


def run(s):
    if own:
        return _own(s)
    op, dtype = s["op"], DTYPES[s["dtype"]]
    if op == "linear":
        return ((s["x"].float() @ _plain_weight(s).t()) * s["scale"]).to(dtype)
    if op == "dgrad":
        return ((s["x"].float() @ _plain_weight(s)) * s["scale"]).to(dtype)
    if op == "act8":
        v, power = _encode8(s["x"], s["format"])
        v = (v * _pow2(power[:, :, None])).view(s["rows"], -1)[:, :s["in"]]
        top = torch.finfo(dtype).max
        return v.clamp(-top, top).to(dtype)
    dw = s["dy"].float().t() @ _plain_values8(s["codes"], s["scales"], s["in"], s["format"])
    dw = dw * 0.5
    if s["add"]:
        dw = dw + s["sum"].float()
    return dw.to(DTYPES[s["grad"]])


def _own(s):
    import odyssey_b200 as ody
    op = s["op"]
    if op in ("linear", "dgrad"):
        w = ody.QuantizedTensor(s["q"], KINDS[s["kind"]][2], s["out"] * s["in"], s["scale"])
        return ody.fp4_linear(s["x"], w) if op == "linear" else ody.fp4_linear_dgrad(s["x"], w)
    if op == "act8":
        return ody.load_activation8(ody.save_activation8(s["x"], s["format"]))
    a = ody.Activation8(s["codes"], s["scales"], s["rows"], s["in"], s["format"])
    return ody.linear_wgrad8(s["dy"], a, alpha=0.5, add=s["sum"] if s["add"] else None, out_dtype=NAMES[s["grad"]])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "act8":
        return _exact_act8(s)
    if case["op"] == "wgrad":
        table = torch.tensor(_grid8(case["format"]), dtype=torch.float64, device=s["codes"].device)
        c = s["codes"].long()
        x = torch.where(c >= 128, -table[c & 127], table[c & 127])
        x = x.view(case["rows"], -1, 32) * _pow2_64(s["scales"].long() - 127)[:, :, None]
        x = x.reshape(case["rows"], -1)[:, :case["in"]]
        dw = 0.5 * torch.einsum("mn,mk->nk", s["dy"].double(), x)
        return dw + s["sum"].double() if case["add"] else dw
    block, size, _ = KINDS[case["kind"]]
    n, k = case["out"], case["in"]
    i = torch.arange(n * k, device=s["q"].device)
    byte = s["q"][(i // block) * size + (i % block) // 2].long()
    code = torch.where(i % 2 == 0, byte // 16, byte % 16)
    mag = code % 8
    value = _pow2_64(mag // 2 - 1) * (1 + 0.5 * (mag % 2).double())
    value = torch.where(mag < 2, mag.double() * (0.5 if case["kind"] == "mxfp4_ocp" else 0.0), value)
    value = torch.where(code >= 8, -value, value)
    scale = s["q"][(i // block) * size + size - 1].long()
    if size == 17:
        value = value * _pow2_64(scale - 127)
    else:
        value = value * torch.tensor(_grid8("e4m3") + [math.nan], dtype=torch.float64, device=i.device)[scale]
    w = value.view(n, k) * s["scale"]
    return torch.einsum("mk,nk->mn" if case["op"] == "linear" else "mn,nk->mk", s["x"].double(), w)


def _grid8(fmt):
    """The non-negative finite values of the format, by code."""
    mant, emin, largest, _, _, _ = FORMATS[fmt]
    found, c = [], 0
    while not found or found[-1] < largest:
        e, m = c >> mant, c % (1 << mant)
        found.append(math.ldexp(m, emin - mant) if e == 0 else math.ldexp((1 << mant) + m, e - 1 + emin - mant))
        c += 1
    return found + ([math.inf] * (127 - len(found)) if len(found) < 127 else [])


def _exact_act8(s):
    """Every value's nearest multiple in its group, found in the list of the format's values; ties to the even code."""
    _, _, largest, _, xmin, xmax = FORMATS[s["format"]]
    grid = [v for v in _grid8(s["format"]) if v < math.inf]
    dev = s["x"].device
    grid = torch.tensor(grid, dtype=torch.float64, device=dev)
    middle = (grid[1:] + grid[:-1]) / 2
    p = _groups(s["x"]).double()
    amax = p.abs().amax(2, keepdim=True)
    power = torch.ceil(torch.log2(amax.clamp(min=1e-300) / largest)).clamp(xmin, xmax)
    # the logarithm may be a step off next to a power of two
    power = torch.where(amax > largest * _pow2_64(power), power + 1, power).clamp(max=xmax)
    power = torch.where((amax <= largest * _pow2_64(power - 1)) & (power > xmin), power - 1, power)
    unit = _pow2_64(power)
    a = p.abs() / unit
    i = torch.searchsorted(middle, a)  # on a tie the lower code; the upper one where that is even
    on_tie = (i < middle.numel()) & (middle[i.clamp(max=middle.numel() - 1)] == a) & (i % 2 == 1)
    v = torch.copysign(grid[i + on_tie.long()] * unit, p).view(s["rows"], -1)[:, :s["in"]]
    top = torch.finfo(s["x"].dtype).max
    return v.clamp(-top, top)
