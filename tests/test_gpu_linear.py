"""The quantised linear layer on the GPU against float64: products with 4-bit
weights, 8-bit activations, the weight gradient, and a training step made of
them."""
import ctypes as C

import numpy as np
import pytest
import torch

import linear_ref as R

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
DTYPES = sorted(DT)
KINDS = sorted(R.W4_KINDS)


@pytest.fixture(scope="module")
def ody():
    import odyssey_b200
    odyssey_b200.lib()
    return odyssey_b200


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(DT[dtype])


def make_w(ody, rng, kind, out, inn):
    q = R.random_weight(rng, R.W4_KINDS[kind], out, inn)
    ts = 0.37 if kind == "nvfp4_tensor" else 1.0
    ts = float(np.float32(ts))
    return ody.QuantizedTensor(dev(q), R.W4_KINDS[kind], out * inn, ts), R.weight(R.W4_KINDS[kind], q, out, inn, ts)


def forward_case(ody, seed, kind, rows, out, inn, dtype, out_dtype=None, dgrad=False, pad=0):
    rng = np.random.default_rng(seed)
    w, w64 = make_w(ody, rng, kind, out, inn)
    cols = out if dgrad else inn
    wide = dev(rng.standard_normal((rows, cols + pad)).astype(np.float32), dtype)
    x = wide[:, pad // 2:pad // 2 + cols]
    y = (ody.fp4_linear_dgrad if dgrad else ody.fp4_linear)(x, w, out_dtype=out_dtype)
    x64, m = R.to64(x), w64 if dgrad else w64.T
    want = x64 @ m
    name = out_dtype or dtype
    assert y.dtype == DT[name] and y.is_cuda
    R.check(y, want, R.tolerance(np.abs(x64) @ np.abs(m), cols, want, name))
    return y


SHAPES = [(1, 1, 1), (1, 16, 32), (2, 33, 7), (32, 120, 400), (5, 84, 120), (32, 10, 84), (1, 256, 1024), (3, 100, 515),
          (8, 128, 256), (9, 257, 1040), (17, 72, 2056), (40, 512, 160), (64, 200, 4608), (65, 129, 96), (130, 300, 258),
          (300, 260, 640), (513, 512, 512)]


@pytest.mark.parametrize("rows,out,inn", SHAPES)
@pytest.mark.parametrize("dgrad", [False, True], ids=["forward", "dgrad"])
def test_product_shapes(ody, rows, out, inn, dgrad):
    for i, kind in enumerate(KINDS):
        for dtype in DTYPES:
            forward_case(ody, rows * 7 + i, kind, rows, out, inn, dtype, dgrad=dgrad)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 15, 16, 17, 31, 32, 33, 47, 64, 66, 100, 128, 129, 255])
def test_product_row_counts(ody, rows):
    for dgrad in (False, True):
        for i, dtype in enumerate(DTYPES):
            forward_case(ody, rows, KINDS[(rows + i) % 4], rows, 336, 768, dtype, dgrad=dgrad)


@pytest.mark.parametrize("inn", [16, 32, 48, 64, 80, 112, 240, 272, 496, 512, 528, 1008, 1024, 1072, 2032, 2048, 2144])
def test_product_block_tails(ody, inn):
    """Widths of whole 16- and 32-element blocks around the kernels' steps."""
    for dgrad in (False, True):
        for kind in KINDS:
            forward_case(ody, inn, kind, 2, 51, inn, "bfloat16", dgrad=dgrad)
            forward_case(ody, inn, kind, 70, 51, inn, "bfloat16", dgrad=dgrad)


# past the one-launch kernels: whole and ragged tiles of the tcgen05 kernel,
# tiles shared by steps, widths of whole blocks and others
LARGE = [(700, 1100, 1030), (2048, 512, 1024), (300, 2500, 1999), (1025, 769, 1568), (64, 4100, 4096), (257, 3000, 4112),
         (4000, 1300, 264)]


@pytest.mark.parametrize("rows,out,inn", LARGE)
@pytest.mark.parametrize("dgrad", [False, True], ids=["forward", "dgrad"])
def test_large_products(ody, rows, out, inn, dgrad):
    for i, (kind, dtype, out_dtype) in enumerate((("nvfp4", "bfloat16", None), ("mxfp4", "float32", None),
                                                  ("mxfp4_ocp", "float16", "float32"), ("nvfp4_tensor", "bfloat16", "float16"))):
        forward_case(ody, rows + i, kind, rows, out, inn, dtype, out_dtype, dgrad, pad=(0, 0, 8, 9)[i])


@pytest.mark.parametrize("rows,out,inn", [(2, 40, 33024), (1, 2500, 10304), (9, 4300, 19072), (3, 70000, 64), (12, 34000, 160)])
@pytest.mark.parametrize("dgrad", [False, True], ids=["forward", "dgrad"])
def test_few_rows_long_reductions(ody, rows, out, inn, dgrad):
    """More than 32 tensor-core steps in a warp's sum, with and without clusters."""
    forward_case(ody, rows, "nvfp4", rows, out, inn, "bfloat16", "float32", dgrad)
    forward_case(ody, rows, "mxfp4", min(rows, 5), out, inn, "float32", None, dgrad)


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_product_types_and_pitches(ody, dtype, out_dtype):
    for dgrad in (False, True):
        for rows, pad in ((2, 24), (2, 7), (90, 16), (90, 5)):
            forward_case(ody, 11, "nvfp4_tensor", rows, 96, 192, dtype, out_dtype, dgrad, pad)


@pytest.mark.parametrize("offset", range(0, 17))
def test_weight_at_any_alignment(ody, offset):
    rng = np.random.default_rng(offset)
    for kind in ("nvfp4", "mxfp4"):
        for inn in (512, 272, 70):
            w, w64 = make_w(ody, rng, kind, 40, inn)
            buf = torch.full((w.data.numel() + 64,), 0x7F, dtype=torch.uint8, device="cuda")
            view = buf[offset:offset + w.data.numel()]
            view.copy_(w.data)
            w = ody.QuantizedTensor(view, w.kind, w.original_numel)
            for rows in (1, 80):
                x = dev(rng.standard_normal((rows, inn)).astype(np.float32), "bfloat16")
                x64 = R.to64(x)
                want = x64 @ w64.T
                R.check(ody.fp4_linear(x, w), want, R.tolerance(np.abs(x64) @ np.abs(w64.T), inn, want, "bfloat16"))
                d = dev(rng.standard_normal((rows, 40)).astype(np.float32), "bfloat16")
                d64 = R.to64(d)
                want = d64 @ w64
                R.check(ody.fp4_linear_dgrad(d, w), want, R.tolerance(np.abs(d64) @ np.abs(w64), 40, want, "bfloat16"))


@pytest.mark.parametrize("overflow", [True, False])
@pytest.mark.parametrize("kind", KINDS)
def test_every_code_and_scale(ody, kind, overflow):
    """One-hot rows read single weights out: every code at every finite scale
    (products with float32 one are exact, so the values are too).  At the two
    largest powers of two 4 x or 6 x the scale passes float32's range: such a
    weight is infinite, and times a zero of the row it makes its results NaN
    as the formula does; without those scales every result is a weight."""
    k = R.W4_KINDS[kind]
    be, sb = R.block(k)
    if sb == 17:
        scales = np.arange(1, 255) if overflow else np.arange(0, 253)
    else:
        scales = np.array([b for b in range(256) if (b & 127) != 127])
    blocks = np.zeros((len(scales), sb), np.uint8)
    blocks[:, :8] = np.arange(16, dtype=np.uint8).reshape(8, 2) @ np.array([16, 1], np.uint8)
    blocks[:, -1] = scales
    n = len(scales)
    w = ody.QuantizedTensor(dev(blocks.reshape(-1)), k, n * be, 1.0)
    want = R.weight(k, blocks, n, be).T
    eye = torch.eye(be, device="cuda")
    with np.errstate(over="ignore"):
        as32 = want.astype(np.float32)
    inf = np.isinf(as32)
    assert inf.any() == (overflow and sb == 17)

    def same(got, values, reached):
        assert np.array_equal(got[~reached], values[~reached]) and not np.isfinite(got[reached]).any()

    for rows in (1, be):
        for r0 in range(0, be, rows):
            got = ody.fp4_linear(eye[r0:r0 + rows], w).cpu().numpy()
            same(got, as32[r0:r0 + rows], np.broadcast_to(inf.any(0), got.shape))
    one = torch.zeros(1, n, device="cuda")
    for j in (0, 1, n // 2, n - 1):
        one.zero_()
        one[0, j] = 1.0
        same(ody.fp4_linear_dgrad(one, w).cpu().numpy()[0], as32[:, j], inf.any(1))


def test_float32_rows_use_all_their_bits(ody):
    """24-bit inputs: a product with one weight per output is exact."""
    rng = np.random.default_rng(5)
    inn = 64
    blocks = np.zeros((inn * inn // 16, 9), np.uint8)
    for r in range(inn):  # W = identity
        e = r * inn + r
        blocks[e // 16, (e % 16) // 2] = 0x20 if e % 2 == 0 else 0x02
    blocks[:, -1] = 56  # 1.0
    w = ody.QuantizedTensor(dev(blocks.reshape(-1)), R.NVFP4, inn * inn)
    for rows in (1, 8, 200, 12000):
        x = rng.standard_normal((rows, inn)).astype(np.float32) * np.exp2(rng.integers(-90, 100, (rows, 1))).astype(np.float32)
        x[:, 3] = np.float32(1.0) + np.float32(2.0 ** -23)
        x[:, 4] = np.finfo(np.float32).max
        for f in (ody.fp4_linear, ody.fp4_linear_dgrad):
            assert np.array_equal(f(dev(x), w).cpu().numpy(), x)
        h = (rng.standard_normal((rows, inn)) * 100).astype(np.float16)
        h[:, 0] = np.float16(65504)
        h[:, 1] = np.float16(6e-8)
        for f in (ody.fp4_linear, ody.fp4_linear_dgrad):
            assert np.array_equal(f(dev(h), w).cpu().numpy(), h)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,inn", [(1, 272), (6, 272), (40, 272), (200, 272), (2000, 4112)])
def test_non_finite_inputs_stay_in_their_row(ody, rows, inn, dtype):
    rng = np.random.default_rng(rows)
    w, w64 = make_w(ody, rng, "nvfp4", 48, inn)
    x = rng.standard_normal((rows, inn)).astype(np.float32)
    bad = rows // 2
    for value in (np.inf, -np.inf, np.nan):
        x[bad, 5] = value
        y = ody.fp4_linear(dev(x, dtype), w).float().cpu().numpy()
        assert np.isfinite(np.delete(y, bad, 0)).all()
        assert not np.isfinite(y[bad][w64[:, 5] != 0]).any()
        g = rng.standard_normal((rows, 48)).astype(np.float32)
        g[bad, 7] = value
        d = ody.fp4_linear_dgrad(dev(g, dtype), w).float().cpu().numpy()
        assert np.isfinite(np.delete(d, bad, 0)).all()
        assert not np.isfinite(d[bad][w64[7] != 0]).any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 100, 9000])
def test_non_finite_block_stays_in_its_results(ody, kind, rows):
    k = R.W4_KINDS[kind]
    be, sb = R.block(k)
    out, inn = 40, 8 * be
    rng = np.random.default_rng(3)
    q = R.random_weight(rng, k, out, inn).reshape(-1, sb)
    q[:, :-1] |= 0x22  # no zero codes
    bad_row, bad_block = 11, 3
    q[bad_row * 8 + bad_block, -1] = 255 if sb == 17 else 0x7F
    w = ody.QuantizedTensor(dev(q.reshape(-1)), k, out * inn)
    x = dev(rng.standard_normal((rows, inn)).astype(np.float32), "bfloat16")
    y = ody.fp4_linear(x, w).float().cpu().numpy()
    assert not np.isfinite(y[:, bad_row]).any() and np.isfinite(np.delete(y, bad_row, 1)).all()
    d = ody.fp4_linear_dgrad(dev(rng.standard_normal((rows, out)).astype(np.float32), "bfloat16"), w)
    d = d.float().cpu().numpy()
    cols = slice(bad_block * be, (bad_block + 1) * be)
    assert not np.isfinite(d[:, cols]).any() and np.isfinite(np.delete(d, np.r_[cols], 1)).all()


def test_agrees_with_dequantize_and_quantize(ody):
    """Weights made by the framework's quantisers, read by its dequantiser."""
    rng = np.random.default_rng(9)
    wf = (rng.standard_normal((96, 224)) * 0.02).astype(np.float32)
    x = dev(rng.standard_normal((12, 224)).astype(np.float32), "bfloat16")
    for to in (ody.to_mxfp4, ody.to_nvfp4, ody.to_nvfp4_tensor_scaled, ody.to_mxfp4_ocp):
        w = to(dev(wf))
        w64, x64 = R.to64(ody.dequantize(w)).reshape(96, 224), R.to64(x)
        want = x64 @ w64.T
        # the dequantiser rounds code x block scale x tensor scale once more
        tol = R.tolerance(np.abs(x64) @ np.abs(w64.T), 224, want, "bfloat16") * (1 + 2.0 ** -22)
        R.check(ody.fp4_linear(x, w), want, tol)


def test_shapes_outputs_and_host_arrays(ody):
    rng = np.random.default_rng(2)
    w, w64 = make_w(ody, rng, "mxfp4", 48, 96)
    x = dev(rng.standard_normal((2, 3, 96)).astype(np.float32))
    y = ody.fp4_linear(x, w)
    assert y.shape == (2, 3, 48)
    out = torch.full((2, 3, 48), 7.0, device="cuda")
    assert ody.fp4_linear(x, w, out=out) is out and torch.equal(out, y)
    assert torch.equal(ody.fp4_linear(x[1, 2], w), y[1, 2])  # a single token without a leading axis
    # columns in another order, a transposed and an expanded input
    xt = x.reshape(6, 96).t().contiguous().t()
    assert torch.equal(ody.fp4_linear(xt, w), y.view(6, 48))
    one = x.reshape(6, 96)[:1]
    assert torch.equal(ody.fp4_linear(one.expand(6, 96), w), ody.fp4_linear(one.repeat(6, 1), w))
    # host arrays: the staged calls give the same bits
    wh = ody.QuantizedTensor(w.data.cpu().numpy(), w.kind, w.original_numel)
    xh = x.cpu().numpy()
    assert np.array_equal(ody.fp4_linear(xh, wh), y.cpu().numpy())
    dy = rng.standard_normal((5, 48)).astype(np.float32)
    assert np.array_equal(ody.fp4_linear_dgrad(dy, wh), ody.fp4_linear_dgrad(dev(dy), w).cpu().numpy())
    a, ah = ody.save_activation8(x), ody.save_activation8(xh)
    assert np.array_equal(a.codes.cpu().numpy(), ah.codes) and np.array_equal(a.scales.cpu().numpy(), ah.scales)
    assert np.array_equal(ody.load_activation8(ah), ody.load_activation8(a).cpu().numpy())
    dy = rng.standard_normal((6, 48)).astype(np.float32)
    base = rng.standard_normal((48, 96)).astype(np.float32)
    got = ody.linear_wgrad8(dy, ah, add=base, alpha=0.5)
    assert np.array_equal(got, ody.linear_wgrad8(dev(dy), a, add=dev(base), alpha=0.5).cpu().numpy())
    buf = base.copy()
    assert ody.linear_wgrad8(dy, ah, add=buf, alpha=0.5, out=buf) is buf and np.array_equal(buf, got)


def test_device_tensor_scale(ody):
    rng = np.random.default_rng(4)
    w, _ = make_w(ody, rng, "nvfp4_tensor", 64, 128)
    x = dev(rng.standard_normal((3, 128)).astype(np.float32))
    wd = ody.QuantizedTensor(w.data, w.kind, w.original_numel, torch.tensor(w.tensor_scale, device="cuda"))
    assert torch.equal(ody.fp4_linear(x, w), ody.fp4_linear(x, wd))
    # the scale of a kind without one is not applied, as in dequantize
    w2 = ody.QuantizedTensor(w.data, R.NVFP4, w.original_numel, 5.0)
    w3 = ody.QuantizedTensor(w.data, R.NVFP4, w.original_numel, 1.0)
    assert torch.equal(ody.fp4_linear(x, w2), ody.fp4_linear(x, w3))


# ---- 8-bit activations ------------------------------------------------------
def save_case(ody, x, fmt):
    """x: CUDA tensor [rows, cols]; codes, scales and restored values exactly."""
    want, power = R.encode8(R.to64(x), fmt)
    a = ody.save_activation8(x, fmt)
    assert np.array_equal(a.scales.cpu().numpy().astype(int) - 127, power)
    codes = a.codes.cpu().numpy()
    rows, cols = x.shape
    dec = (R.e4m3 if fmt == "e4m3" else R.e5m2)(codes) * np.repeat(2.0 ** power, 32, 1)
    assert np.array_equal(dec[:, :cols], want, equal_nan=True) and not codes[:, cols:].any()
    got = R.to64(ody.load_activation8(a, "float32"))
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(R.to64(ody.load_activation8(a, "bfloat16")), want, equal_nan=True)
    with np.errstate(over="ignore"):
        h = np.where(np.isfinite(want), np.clip(want, -65504, 65504), want).astype(np.float16)
    assert np.array_equal(ody.load_activation8(a, "float16").cpu().numpy(), h, equal_nan=True)
    return a, want


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (7, 100), (33, 257), (130, 1000), (64, 4096)])
def test_activation8_shapes(ody, rows, cols, dtype, fmt):
    rng = np.random.default_rng(rows * cols)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 9, (rows, 1)))
    save_case(ody, dev(x.astype(np.float32), dtype), fmt)
    wide = dev(np.pad(x, ((0, 0), (3, 4))).astype(np.float32), dtype)
    save_case(ody, wide[:, 3:3 + cols], fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_activation8_every_rounding(ody, fmt):
    """Every value of the format, every middle of two, and their neighbours in
    float32, at scales across float32's range (the group's largest element
    pins the power of two)."""
    grid = (R.e4m3 if fmt == "e4m3" else R.e5m2)(np.arange(0x7F if fmt == "e4m3" else 0x7C))
    mid = (grid[1:] + grid[:-1]) / 2
    v = np.concatenate([grid, mid]).astype(np.float32)
    v = np.concatenate([v, np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(0))])
    v = np.minimum(v, np.float32(grid[-1]))
    v = np.resize(v, -(-len(v) // 31) * 31).reshape(-1, 31)
    v = np.concatenate([v, np.full((len(v), 1), grid[-1], np.float32)], 1).reshape(1, -1)
    v[:, ::3] *= -1
    lo, hi = (-117, 119) if fmt == "e4m3" else (-110, 112)
    for p in (lo, lo + 1, -60, -1, 0, 1, 60, hi):
        save_case(ody, dev((v * np.float32(2.0) ** p).astype(np.float32)), fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_activation8_special_values(ody, dtype, fmt):
    t = torch.finfo(DT[dtype])
    x = torch.zeros(12, 32, dtype=DT[dtype], device="cuda")
    x[1, 0] = -0.0
    x[2] = t.max
    x[3, 4], x[3, 5] = -t.max, 1.0
    x[4, 9] = t.smallest_normal
    x[5, 9] = t.smallest_normal / 4  # subnormal
    x[6, 1], x[6, 2], x[6, 3] = float("inf"), float("-inf"), 2.5
    x[7, 1], x[7, 2] = float("nan"), -3.0
    x[8] = float("nan")
    x[9] = float("inf")
    x[10, :2] = torch.tensor([448.0, 449.0])
    x[11, :2] = torch.tensor([57344.0, -60000.0])
    a, _ = save_case(ody, x, fmt)
    assert not torch.isfinite(ody.load_activation8(a)[[6, 6, 7, 9], [1, 2, 1, 31]]).any()


# ---- weight gradient --------------------------------------------------------
def wgrad_case(ody, seed, rows, out, inn, dtype, out_dtype, fmt="e4m3", add=False, alpha=1.0, pad=0):
    rng = np.random.default_rng(seed)
    a = ody.save_activation8(dev((rng.standard_normal((rows, inn)) * np.exp2(rng.integers(-3, 4, (rows, 1)))).astype(np.float32)),
                             fmt)
    dy = dev(rng.standard_normal((rows, out + pad)).astype(np.float32), dtype)[:, pad // 2:pad // 2 + out]
    base = dev(rng.standard_normal((out, inn)).astype(np.float32), out_dtype) if add else None
    dw = ody.linear_wgrad8(dy, a, add=base, alpha=alpha, out_dtype=out_dtype)
    assert dw.dtype == DT[out_dtype]
    d64, x64 = R.to64(dy), R.to64(ody.load_activation8(a, "float32"))
    want = alpha * (d64.T @ x64)
    terms = abs(alpha) * (np.abs(d64.T) @ np.abs(x64))
    if add:
        want, terms = want + R.to64(base), terms + np.abs(R.to64(base))
    R.check(dw, want, R.tolerance(terms, rows, want, out_dtype))


@pytest.mark.parametrize("rows,out,inn", [(1, 1, 1), (1, 8, 32), (2, 3, 5), (7, 40, 33), (32, 120, 400), (64, 128, 256),
                                          (65, 100, 515), (130, 257, 96), (333, 72, 160), (1000, 64, 64), (1500, 10, 84),
                                          (4100, 33, 70), (512, 512, 512)])
def test_wgrad_shapes(ody, rows, out, inn):
    for fmt in ("e4m3", "e5m2"):
        for dtype in DTYPES:
            wgrad_case(ody, rows, rows, out, inn, dtype, "float32", fmt)
            wgrad_case(ody, rows, rows, out, inn, dtype, dtype, fmt, add=True, alpha=0.25)


@pytest.mark.parametrize("rows,out,inn", [(1500, 1100, 1030), (20000, 64, 64), (700, 2048, 1000), (3001, 520, 1313),
                                          (4096, 1024, 512)])
def test_large_wgrads(ody, rows, out, inn):
    for i, (fmt, dtype, out_dtype) in enumerate((("e4m3", "bfloat16", "bfloat16"), ("e5m2", "float16", "float32"),
                                                 ("e4m3", "float32", "float32"), ("e4m3", "bfloat16", "float16"))):
        wgrad_case(ody, rows + i, rows, out, inn, dtype, out_dtype, fmt, add=i % 2 == 1, alpha=0.5, pad=(0, 0, 0, 9)[i])


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_wgrad_types_and_pitches(ody, dtype, out_dtype):
    for pad in (0, 16, 7):
        for add in (False, True):
            wgrad_case(ody, 21, 200, 136, 224, dtype, out_dtype, add=add, alpha=-0.5, pad=pad)


def test_wgrad_accumulates_in_place(ody):
    rng = np.random.default_rng(1)
    a = ody.save_activation8(dev(rng.standard_normal((50, 64)).astype(np.float32)))
    dy = dev(rng.standard_normal((50, 96)).astype(np.float32))
    base = torch.randn(96, 64, device="cuda")
    want = ody.linear_wgrad8(dy, a, add=base)
    got = base.clone()
    assert ody.linear_wgrad8(dy, a, add=got, out=got) is got and torch.equal(got, want)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_wgrad_passes_non_finite_on(ody, fmt):
    """An infinity or NaN of the activation or of dy reaches its gradients and
    no others, so the step's finite check sees it."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((70, 96)).astype(np.float32)
    x[33, 40] = np.inf
    dy = rng.standard_normal((70, 48)).astype(np.float32)
    dw = ody.linear_wgrad8(dev(dy, "bfloat16"), ody.save_activation8(dev(x), fmt)).float().cpu().numpy()
    assert not np.isfinite(dw[:, 40]).any() and np.isfinite(np.delete(dw, 40, 1)).all()
    x[33, 40] = 1.0
    for dtype in DTYPES:
        for v in (np.inf, np.nan):
            dy[5, 6] = v
            dw = ody.linear_wgrad8(dev(dy, dtype), ody.save_activation8(dev(x), fmt)).float().cpu().numpy()
            assert not np.isfinite(dw[6]).any() and np.isfinite(np.delete(dw, 6, 0)).all()


def test_gradients_against_differences(ody):
    """dx and dW of L = sum(y * g) against central differences in float64 of
    the forward formula with the same weights and the restored activation."""
    rng = np.random.default_rng(12)
    w, w64 = make_w(ody, rng, "nvfp4", 24, 48)
    a = ody.save_activation8(dev(rng.standard_normal((6, 48)).astype(np.float32)))
    x64 = R.to64(ody.load_activation8(a, "float32"))
    g = rng.standard_normal((6, 24)).astype(np.float32)
    dx = R.to64(ody.fp4_linear_dgrad(dev(g), w))
    dw = R.to64(ody.linear_wgrad8(dev(g), a))
    g64 = g.astype(np.float64)

    def loss(x, w):
        return float((x @ w.T * g64).sum())

    h = 2.0 ** -10  # L is bilinear: central differences are exact up to float64 rounding
    for i, j in ((0, 0), (2, 17), (5, 47)):
        e = np.zeros_like(x64)
        e[i, j] = h
        d = (loss(x64 + e, w64) - loss(x64 - e, w64)) / (2 * h)
        assert abs(d - dx[i, j]) <= 2.0 ** -17 * (np.abs(g64[i]) @ np.abs(w64[:, j])) + 1e-8
    for i, j in ((0, 0), (11, 30), (23, 47)):
        e = np.zeros_like(w64)
        e[i, j] = h
        d = (loss(x64, w64 + e) - loss(x64, w64 - e)) / (2 * h)
        assert abs(d - dw[i, j]) <= 2.0 ** -17 * (np.abs(g64[:, i]) @ np.abs(x64[:, j])) + 1e-8


# ---- streams, graphs, repeats, neighbours -----------------------------------
def test_same_call_same_bits(ody):
    rng = np.random.default_rng(6)
    for rows, out, inn in ((1, 512, 1024), (8, 500, 528), (300, 256, 2048), (2000, 96, 160), (1111, 1300, 1040)):
        w, _ = make_w(ody, rng, "nvfp4", out, inn)
        x = dev(rng.standard_normal((rows, inn)).astype(np.float32))
        dy = dev(rng.standard_normal((rows, out)).astype(np.float32), "bfloat16")
        a = ody.save_activation8(x)
        first = (ody.fp4_linear(x, w), ody.fp4_linear_dgrad(dy, w), ody.linear_wgrad8(dy, a, out_dtype="float32"))
        for _ in range(3):
            for f, s in zip(first, (ody.fp4_linear(x, w), ody.fp4_linear_dgrad(dy, w),
                                    ody.linear_wgrad8(dy, a, out_dtype="float32"))):
                assert torch.equal(f, s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_do_not_depend_on_each_other(ody, dtype):
    """Among few rows a row's results are the same bits whatever their number."""
    rng = np.random.default_rng(21)
    parts = {"bfloat16": 1, "float16": 2, "float32": 3}[dtype]
    for out, inn in ((72, 1056), (600, 64), (1030, 2080)):
        w, _ = make_w(ody, rng, "mxfp4", out, inn)
        for fn, cols, most in ((ody.fp4_linear, inn, 32 // parts), (ody.fp4_linear_dgrad, out, 16 // parts)):
            x = dev(rng.standard_normal((most, cols)).astype(np.float32), dtype)
            whole = fn(x, w)
            for n in (1, 2, 8 // parts, 8 // parts + 1):
                assert torch.equal(fn(x[:n], w), whole[:n]), (out, inn, n)
            assert torch.equal(fn(x[-1:], w), whole[-1:])


def test_captured_and_replayed_on_side_streams(ody):
    """Two captured layers of different sizes, replayed at once on two streams
    with new inputs, give the bits of eager calls."""
    rng = np.random.default_rng(7)
    sets = []
    for rows, out, inn in ((900, 1100, 1040), (200, 384, 640), (3, 257, 1040)):
        w, _ = make_w(ody, rng, "mxfp4", out, inn)
        x = dev(rng.standard_normal((rows, inn)).astype(np.float32), "bfloat16")
        dy = dev(rng.standard_normal((rows, out)).astype(np.float32), "bfloat16")
        sets.append([w, x, dy])

    def layer(w, x, dy):
        y = ody.fp4_linear(x, w)
        a = ody.save_activation8(x)
        return y, ody.fp4_linear_dgrad(dy, w), ody.linear_wgrad8(dy, a, out_dtype="float32")

    graphs = []
    for s in sets:
        layer(*s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = layer(*s)
        graphs.append((g, res))
    streams = [torch.cuda.Stream() for _ in sets]
    for rep in range(3):
        for s in sets:
            s[1].copy_(torch.randn_like(s[1]))
            s[2].copy_(torch.randn_like(s[2]))
        torch.cuda.synchronize()
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, (_, res) in zip(sets, graphs):
            for got, want in zip(res, layer(*s)):
                assert torch.equal(got, want)


def test_overlapping_calls_on_two_streams(ody):
    rng = np.random.default_rng(17)
    w, _ = make_w(ody, rng, "nvfp4", 1500, 768)
    xs = [dev(rng.standard_normal((950, 768)).astype(np.float32)) for _ in range(2)]
    want = [ody.fp4_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ody.fp4_linear(xs[i], w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("rows,out,inn", [(1, 72, 144), (5, 72, 144), (70, 72, 144), (300, 72, 144), (500, 1503, 1552)])
def test_pitched_outputs_leave_their_neighbours(ody, rows, out, inn):
    """The stream forms write rows x columns of the output and nothing else,
    with float16, bfloat16 and float32 results at odd pitches."""
    from odyssey_b200 import _lib as L
    lib = L.lib()
    rng = np.random.default_rng(rows)
    w, w64 = make_w(ody, rng, "mxfp4", out, inn)
    st = torch.cuda.current_stream().cuda_stream
    for op, cols, width in ((L.LINEAR_FORWARD, inn, out), (L.LINEAR_DGRAD, out, inn)):
        x = dev(rng.standard_normal((rows, cols)).astype(np.float32))
        x64 = R.to64(x)
        m = w64.T if op == L.LINEAR_FORWARD else w64
        want = x64 @ m
        for code, name in ((L.F32, "float32"), (L.F16, "float16"), (L.BF16, "bfloat16")):
            for ld in (width + 8, width + 5):
                buf = torch.full((rows + 2, ld), 77.0, dtype=DT[name], device="cuda")
                n = lib.ody_linear_workspace(op, rows, out, inn, L.F32)
                ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
                fn = lib.ody_fp4_linear_on_stream if op == L.LINEAR_FORWARD else lib.ody_fp4_linear_dgrad_on_stream
                L.check(fn(w.kind, w.data.data_ptr(), None, 1.0, out, inn, x.data_ptr(), L.F32, rows, cols,
                           buf[1:].data_ptr(), code, ld, ws.data_ptr(), n, st))
                R.check(buf[1:rows + 1, :width], want, R.tolerance(np.abs(x64) @ np.abs(m), cols, want, name))
                assert (buf[0] == 77).all() and (buf[rows + 1] == 77).all() and (buf[1:rows + 1, width:] == 77).all()


def test_activation_load_leaves_its_neighbours(ody):
    from odyssey_b200 import _lib as L
    a = ody.save_activation8(torch.randn(5, 45, device="cuda"))
    for code, name in ((L.F32, "float32"), (L.F16, "float16"), (L.BF16, "bfloat16")):
        for ld in (48, 51):
            buf = torch.full((7, ld), 77.0, dtype=DT[name], device="cuda")
            L.check(L.lib().ody_act8_load_on_stream(L.A8_E4M3, a.codes.data_ptr(), a.scales.data_ptr(), 5, 45,
                                                    buf[1:].data_ptr(), code, ld, torch.cuda.current_stream().cuda_stream))
            assert torch.equal(buf[1:6, :45], ody.load_activation8(a, name))
            assert (buf[0] == 77).all() and (buf[6] == 77).all() and (buf[1:6, 45:] == 77).all()


def test_wait_that_runs_out_is_reported(ody):
    """A device-side wait for something that never comes ends after its limit
    (about 20 ms here), the next query reports it once, and the layer still works."""
    from odyssey_b200 import _lib as L
    ody.linear_status()
    st = torch.cuda.current_stream().cuda_stream
    hook = L.lib().odyx_linear_wait_selftest
    hook.argtypes = [C.c_int64, C.c_void_p]
    assert hook(40_000_000, st) == 0
    with pytest.raises(ody.OdysseyError, match="ran out") as e:
        ody.linear_status()
    assert e.value.code == L.ERR_DEVICE_BOUNDS
    ody.linear_status()
    forward_case(ody, 1, "nvfp4", 300, 256, 512, "bfloat16")


def test_first_calls_of_a_process_inside_a_capture(tmp_path):
    """No call before the capture: kernels, attributes and tensor maps are set
    up while the stream is being captured."""
    import os
    import subprocess
    import sys
    code = """
import torch, odyssey_b200 as ody
w = ody.QuantizedTensor(torch.zeros(1100 * 1040 // 16 * 9, dtype=torch.uint8, device="cuda"), 7, 1100 * 1040)
w.data.random_(0, 120, generator=torch.Generator(device="cuda").manual_seed(1))
xs = [torch.randn(r, 1040, device="cuda") for r in (1, 40, 900)]
dys = [torch.randn(r, 1100, device="cuda") for r in (1, 40, 900)]
torch.cuda.synchronize()
def layer():
    res = []
    for x, dy in zip(xs, dys):
        a = ody.save_activation8(x)
        res += [ody.fp4_linear(x, w), ody.fp4_linear_dgrad(dy, w), ody.linear_wgrad8(dy, a), ody.load_activation8(a)]
    return res
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    res = layer()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(res, layer()))
ody.linear_status()
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stdout + r.stderr


def test_refusals_on_device_memory(ody):
    """What only shows with device pointers: host memory among them, unaligned
    buffers, a workspace that is missing, too small or unaligned; nothing is
    launched and the output stays as it was."""
    from odyssey_b200 import _lib as L
    lib = L.lib()
    rng = np.random.default_rng(0)
    w, _ = make_w(ody, rng, "nvfp4", 1100, 1040)
    x = torch.randn(900, 1040, device="cuda")
    y = torch.full((900, 1100), 5.0, device="cuda")
    need = lib.ody_linear_workspace(L.LINEAR_FORWARD, 900, 1100, 1040, L.F32)
    assert need > 0
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    host = np.zeros(900 * 1100, np.float32)

    def call(q=w.data.data_ptr(), x=x.data_ptr(), y=y.data_ptr(), ts=None, ws=ws.data_ptr(), n=need):
        return lib.ody_fp4_linear_on_stream(w.kind, q, ts, 1.0, 1100, 1040, x, L.F32, 900, 1040, y, L.F32, 1100, ws, n, st)

    assert call(ws=None) == L.ERR_ARG and call(n=need - 1) == L.ERR_ARG and call(ws=ws.data_ptr() + 16) == L.ERR_ARG
    assert call(x=host.ctypes.data) == L.ERR_ARG and call(y=host.ctypes.data) == L.ERR_ARG
    assert call(ts=host.ctypes.data) == L.ERR_ARG and call(ws=host.ctypes.data) == L.ERR_ARG
    assert call(x=x.data_ptr() + 2) == L.ERR_ARG and call(y=y.data_ptr() + 1) == L.ERR_ARG
    scale = torch.ones(2, device="cuda")
    assert call(ts=scale.data_ptr() + 2) == L.ERR_ARG
    assert call(y=x.data_ptr()) == L.ERR_ARG and call(y=w.data.data_ptr()) == L.ERR_ARG
    torch.cuda.synchronize()
    assert (y == 5.0).all()
    assert call() == L.OK
    ody.linear_status()
    assert torch.equal(y, ody.fp4_linear(x, w))
    a = ody.save_activation8(x)
    shifted = torch.empty(a.codes.numel() + 8, dtype=torch.uint8, device="cuda")[8:]
    with pytest.raises(ody.OdysseyError, match="16-byte aligned"):
        ody.load_activation8(ody.Activation8(shifted.view(900, -1), a.scales, 900, 1040))
    with pytest.raises(ody.OdysseyError, match="one device"):
        ody.linear_wgrad8(torch.randn(900, 8), a)
    with pytest.raises(ody.OdysseyError, match="one device"):
        ody.fp4_linear(x.cpu(), w)
    with pytest.raises(ody.OdysseyError, match="one float32"):
        ody.fp4_linear(x, ody.QuantizedTensor(w.data, R.NVFP4_TENSOR, w.original_numel, torch.ones(2, device="cuda")))


# ---- offsets past 32 bits ---------------------------------------------------
def test_weight_of_more_than_2_32_elements(ody):
    out, inn = 70001, 65536
    gen = torch.Generator(device="cuda").manual_seed(3)
    n = out * inn // 16
    blocks = torch.randint(0, 256, (n, 9), dtype=torch.uint8, device="cuda", generator=gen)
    blocks[:, 8] = 48
    w = ody.QuantizedTensor(blocks.view(-1), R.NVFP4, out * inn)
    x = torch.randn(2, inn, device="cuda", generator=gen).bfloat16()
    y = ody.fp4_linear(x, w)
    rows = [0, 1, 32767, 32768, 65535, 65536, 70000]
    per = inn // 16
    w64 = np.stack([R.weight(R.NVFP4, blocks[r * per:(r + 1) * per].cpu().numpy(), 1, inn)[0] for r in rows])
    x64 = R.to64(x)
    want = x64 @ w64.T
    R.check(y[:, rows], want, R.tolerance(np.abs(x64) @ np.abs(w64.T), inn, want, "bfloat16"))
    dy = torch.zeros(1, out, device="cuda")
    dy[0, rows] = torch.randn(len(rows), device="cuda", generator=gen)
    d64 = R.to64(dy[:, rows])
    want = d64 @ w64
    R.check(ody.fp4_linear_dgrad(dy, w), want, R.tolerance(np.abs(d64) @ np.abs(w64), out, want, "float32"))


def test_rows_of_more_than_2_32_bytes(ody):
    """float32 features whose place in a row passes 32 bits: only the last 64
    count (all other weights are zero), and the first 64 are large."""
    inn, out = 2**30 + 64, 8
    data = torch.zeros(out, inn // 32, 17, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(7)
    last = rng.integers(0, 256, (out, 2, 17), dtype=np.uint8)
    last[:, :, -1] = 127
    data[:, -2:] = torch.from_numpy(last).cuda()
    x = torch.zeros(1, inn, device="cuda")
    x[0, :64] = 1e6
    x[0, -64:] = torch.from_numpy(rng.standard_normal(64).astype(np.float32)).cuda()
    w = ody.QuantizedTensor(data.view(-1), R.MXFP4, out * inn)
    m = R.weight(R.MXFP4, last.reshape(-1), out, 64)
    x64 = R.to64(x[:, -64:])
    R.check(ody.fp4_linear(x, w), x64 @ m.T, R.tolerance(np.abs(x64) @ np.abs(m.T), 64, x64 @ m.T, "float32"))


def test_activation_of_more_than_2_32_elements(ody):
    rows, cols = 1 << 20, 4160
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    a = ody.save_activation8(x)
    back = ody.load_activation8(a)
    at = [0, 1, 500000, 1032443, 1032444, rows - 1]  # 2^32 / 4160 = 1032444.06
    want, power = R.encode8(R.to64(x[at]), "e4m3")
    assert np.array_equal(a.scales[at].cpu().numpy().astype(int) - 127, power)
    assert np.array_equal(R.to64(back[at]), want)
    del back
    dy = torch.zeros(rows, 16, dtype=torch.bfloat16, device="cuda")
    dy[at] = torch.randn(len(at), 16, device="cuda").bfloat16()
    d64 = R.to64(dy[at])
    want_dw = d64.T @ want
    dw = ody.linear_wgrad8(dy, a, out_dtype="float32")
    R.check(dw, want_dw, R.tolerance(np.abs(d64.T) @ np.abs(want), rows, want_dw, "float32"))


# ---- together ---------------------------------------------------------------
def test_training_step_through_the_layer(ody):
    """Two linear layers trained from the step's own codes: forward through the
    4-bit weights, 8-bit activations, both gradients, and the step that takes
    them; every piece against float64, and the step's skip on an overflow."""
    from odyssey_b200 import _lib as L
    rng = np.random.default_rng(31)
    shapes = [(96, 160), (64, 96)]
    scale = 1024.0
    ctx = ody.MixedPrecisionStep([o * i for o, i in shapes], grad_dtype="bfloat16", quant="nvfp4_tensor", optimizer="adamw",
                                 learning_rate=1e-3, initial_scale=scale)
    for i, (o, n) in enumerate(shapes):
        ctx.set_master(i, (rng.standard_normal(o * n) * 0.05).astype(np.float32))
    # a step with zero gradients leaves the masters and makes the first codes
    for i, (o, n) in enumerate(shapes):
        ctx.set_grad(i, torch.zeros(o * n, dtype=torch.bfloat16, device="cuda"))
    ctx.step(1)

    def codes(i):
        buf = torch.empty(L.quant_bytes(L.Q_NVFP4_TENSOR, ctx.numels[i]), dtype=torch.uint8, device="cuda")
        return ctx.get_quant(i, buf)

    x = dev(rng.standard_normal((48, 160)).astype(np.float32), "bfloat16")
    for t in range(2, 5):
        w = [codes(0), codes(1)]
        w64 = [R.weight(R.NVFP4_TENSOR, q.data.cpu().numpy(), *s, q.tensor_scale) for q, s in zip(w, shapes)]
        a0 = ody.save_activation8(x)
        h = ody.fp4_linear(x, w[0])
        a1 = ody.save_activation8(h, "e5m2")
        y = ody.fp4_linear(h, w[1], out_dtype="float32")
        x64, h64 = R.to64(x), R.to64(h)
        R.check(h, x64 @ w64[0].T, R.tolerance(np.abs(x64) @ np.abs(w64[0].T), 160, x64 @ w64[0].T, "bfloat16"))
        R.check(y, h64 @ w64[1].T, R.tolerance(np.abs(h64) @ np.abs(w64[1].T), 96, h64 @ w64[1].T, "float32"))
        dy = (y * (2 * scale / y.numel())).bfloat16()  # gradient of scale * mean(y^2)
        if t == 4:
            dy[3, 5] = float("inf")
        dw1 = ody.linear_wgrad8(dy, a1)
        dh = ody.fp4_linear_dgrad(dy, w[1])
        dw0 = ody.linear_wgrad8(dh, a0)
        if t < 4:
            d64, hr = R.to64(dy), R.to64(ody.load_activation8(a1))
            R.check(dw1, d64.T @ hr, R.tolerance(np.abs(d64.T) @ np.abs(hr), 48, d64.T @ hr, "bfloat16"))
            R.check(dh, d64 @ w64[1], R.tolerance(np.abs(d64) @ np.abs(w64[1]), 64, d64 @ w64[1], "bfloat16"))
            g64, xr = R.to64(dh), R.to64(ody.load_activation8(a0))
            R.check(dw0, g64.T @ xr, R.tolerance(np.abs(g64.T) @ np.abs(xr), 48, g64.T @ xr, "bfloat16"))
        before = ctx.master(0).copy()
        ctx.set_grad(0, dw0)
        ctx.set_grad(1, dw1)
        r = ctx.step(t)
        assert bool(r["skipped"]) == (t == 4)
        assert np.array_equal(before, ctx.master(0)) == (t == 4)
    ctx.close()
