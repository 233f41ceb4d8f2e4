"""Plain float64 statements of the quantised linear layer, for its tests."""
import numpy as np

MXFP4, NVFP4, NVFP4_TENSOR, MXFP4_OCP = 6, 7, 8, 9
W4_KINDS = {"mxfp4": MXFP4, "nvfp4": NVFP4, "nvfp4_tensor": NVFP4_TENSOR, "mxfp4_ocp": MXFP4_OCP}
GROUP = 32


def block(kind):
    """(elements, bytes) of one block."""
    return (32, 17) if kind in (MXFP4, MXFP4_OCP) else (16, 9)


def e4m3(byte):
    b = np.asarray(byte, np.int64)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >= 128, -v, v)


def e5m2(byte):
    b = np.asarray(byte, np.int64)
    e, m = (b >> 2) & 31, b & 3
    v = np.where(e == 0, m * 2.0 ** -16, (4 + m) * 2.0 ** (e - 17.0))
    v = np.where(e == 31, np.where(m == 0, np.inf, np.nan), v)
    return np.where(b >= 128, -v, v)


def weight(kind, q, out, inn, tensor_scale=1.0):
    """W [out, in] in float64 from its bytes."""
    be, sb = block(kind)
    b = np.asarray(q, np.uint8).reshape(-1, sb)
    codes = np.stack([b[:, :-1] >> 4, b[:, :-1] & 15], 2).reshape(-1, be)
    half = 0.5 if kind == MXFP4_OCP else 0.0
    mag = np.array([0, half, 1, 1.5, 2, 3, 4, 6])[codes & 7]
    byte = b[:, -1].astype(np.float64)
    if kind == MXFP4_OCP:
        scale = np.where(byte == 255, np.nan, 2.0 ** (byte - 127))
    elif kind == MXFP4:
        scale = np.where(byte == 255, np.inf, np.where(byte == 0, 0.0, 2.0 ** (byte - 127)))
    else:
        scale = e4m3(b[:, -1])
    with np.errstate(invalid="ignore"):
        v = np.where(mag == 0, 0.0, mag * scale[:, None]) if kind != MXFP4_OCP else mag * scale[:, None]
    v = np.where(codes >= 8, -v, v).reshape(-1)[:out * inn].reshape(out, inn)
    return v * (tensor_scale if kind == NVFP4_TENSOR else 1.0)


def random_weight(rng, kind, out, inn, spread=4):
    """Bytes of a weight with random codes and block scales around one."""
    be, sb = block(kind)
    n = -(-out * inn // be)
    b = rng.integers(0, 256, (n, sb), dtype=np.uint8)
    if kind in (MXFP4, MXFP4_OCP):
        b[:, -1] = rng.integers(127 - spread, 127 + spread + 1, n)
    else:
        b[:, -1] = rng.integers(56 - 8 * spread, 56 + 8 * spread, n)
    return b.reshape(-1)


def to64(x):
    """float64 values of a torch tensor or numpy array."""
    return x.detach().double().cpu().numpy() if hasattr(x, "detach") else np.asarray(x, np.float64)


def encode8(x, fmt):
    """(values the codes stand for, power of two per group) of float64 rows x,
    by the definition and with every step exact in float64."""
    largest, mant, emin, xmin, xmax = (448.0, 3, -6, -117, 119) if fmt == "e4m3" else (57344.0, 2, -14, -110, 112)
    rows, cols = x.shape
    g = -(-cols // GROUP)
    p = np.zeros((rows, g * GROUP))
    p[:, :cols] = x
    p = p.reshape(rows, g, GROUP)
    amax = np.where(np.isfinite(p), np.abs(p), 0.0).max(2)
    power = np.full(amax.shape, xmin)
    while True:  # the least power in range that holds the largest finite element
        more = (amax > largest * 2.0 ** power) & (power < xmax)
        if not more.any():
            break
        power = power + more
    with np.errstate(invalid="ignore"):
        v = p / 2.0 ** power[:, :, None]
        e = np.floor(np.log2(np.maximum(np.abs(np.where(np.isfinite(v), v, 0.0)), 2.0 ** emin)))
        e = np.where(2.0 ** (e + 1) <= np.abs(v), e + 1, np.where(2.0 ** e > np.maximum(np.abs(v), 2.0 ** emin), e - 1, e))
        step = 2.0 ** (e - mant)
        r = np.clip(np.round(v / step) * step, -largest, largest)
    r = np.where(np.isnan(p), np.nan, np.where(np.isinf(p), p if fmt == "e5m2" else np.nan, r))
    return (r * 2.0 ** power[:, :, None]).reshape(rows, -1)[:, :cols], power


HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}  # half the least subnormal


def tolerance(terms, reduction, value, dtype):
    """Elementwise bound on a product's error.  Every product is exact; a sum
    in float32 of `reduction` of them is taken in at most 32 + reduction / 256
    additions that each lose at most 2^-22 of the sum of magnitudes `terms`
    (a tensor core cuts aligned products off rather than rounding them, at
    2^-23 of the largest or better, 16 at a time; the float32 pipe's 64 +
    reduction / 64 additions lose 2^-24 each, which is less).  Then two
    roundings of the scale in float32, and half a step of the output."""
    acc = terms * (2.0 ** -22 * (32 + reduction / 256) + 2.0 ** -23)
    return acc + (np.abs(value) + acc) * HALF_STEP[dtype] + TINY[dtype]


def check(got, want, tol):
    """Finite results within tol; where the formula is not finite, no finite one."""
    got = to64(got)
    assert got.shape == want.shape, (got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine), "finite and non-finite results are not where the formula's are"
    bad = fine & ~(np.abs(np.where(fine, got - want, 0.0)) <= np.where(fine, tol, 0.0))
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.size} off; first at {i}: {got[i]!r}, expected {want[i]!r} "
                             f"within {tol[i]!r}")
