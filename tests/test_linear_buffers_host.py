"""What the quantised linear layer's Python calls hand to the library, and the
buffers that they refuse, without a GPU."""
import ctypes as C
import types
import weakref

import numpy as np
import pytest


@pytest.fixture(scope="module")
def ody():
    from odyssey_b200.build import build
    build()
    import odyssey_b200
    odyssey_b200.lib()
    return odyssey_b200


def refused(ody, code, match, fn, *args, **kw):
    with pytest.raises(ody.OdysseyError, match=match) as e:
        fn(*args, **kw)
    assert e.value.code == code


def weight(ody, out, inn, kind=7):
    from odyssey_b200 import _lib as L
    return ody.QuantizedTensor(np.zeros(L.quant_bytes(kind, out * inn), np.uint8), kind, out * inn)


@pytest.mark.parametrize("name", ["fp4_linear", "fp4_linear_dgrad"])
@pytest.mark.parametrize("torch_weight", [False, True])
def test_strided_host_weight_lives_until_the_call_is_done(ody, monkeypatch, name, torch_weight):
    """A weight that is not contiguous is copied; the copy is what the library
    reads, so it is still there, with the weight's bytes, when it does."""
    import torch
    from odyssey_b200 import linear, _lib as L
    out, inn = 512, 512
    n = L.quant_bytes(L.Q_NVFP4, out * inn)
    wide = np.random.default_rng(1).integers(0, 256, 2 * n, dtype=np.uint8)
    want = wide[::2].tobytes()
    data = torch.from_numpy(wide)[::2] if torch_weight else wide[::2]
    copies, seen = [], []
    contiguous = L.contiguous

    def tracked(x):
        c = contiguous(x)
        copies.append(weakref.ref(c))
        return c

    def entry(kind, q, *rest):
        decoys = [np.full(n, 0xEE, np.uint8) for _ in range(4)]  # what a freed copy's memory would be given to
        seen.append((C.string_at(q, n) == want, [c() is not None for c in copies]))
        return len(decoys) - 4

    monkeypatch.setattr(linear.L, "contiguous", tracked)
    monkeypatch.setattr(linear.L, "lib", lambda: types.SimpleNamespace(**{"ody_" + name: entry}))
    w = ody.QuantizedTensor(data, L.Q_NVFP4, out * inn)
    getattr(ody, name)(np.ones((2, 512), np.float32), w)
    assert seen == [(True, [True])]


def test_load_refuses_a_shape_of_other_elements(ody):
    """The shape an Activation8 carries sizes the result, so it has to hold the
    rows and columns that are written there: not fewer (a write past the
    buffer), not more (an unwritten rest)."""
    from odyssey_b200 import _lib as L
    codes, scales = np.zeros((3, 64), np.uint8), np.zeros((3, 2), np.uint8)
    for shape in ((2, 40), (3, 39), (40,), (), (0, 40), (4, 40), (3, 41), (2, 3, 40)):
        a = ody.Activation8(codes, scales, 3, 40, shape=shape)
        refused(ody, L.ERR_SHAPE, "120 elements", ody.load_activation8, a)
        refused(ody, L.ERR_SHAPE, "120 elements", ody.load_activation8, a, out=np.empty(shape, np.float32), dtype="float32")


def test_results_that_are_operands_are_refused(ody):
    """By name of the caller's buffers, before anything is copied or launched."""
    from odyssey_b200 import _lib as L
    import torch
    n = 32
    w = ody.QuantizedTensor(np.zeros(L.quant_bytes(L.Q_NVFP4, n * n), np.uint8), L.Q_NVFP4, n * n)
    x = np.ones((n, n), np.float32)
    for fn in (ody.fp4_linear, ody.fp4_linear_dgrad):
        refused(ody, L.ERR_ARG, "must not be or overlap an operand", fn, x, w, out=x)
        t = torch.ones(n, n)
        refused(ody, L.ERR_ARG, "must not be or overlap an operand", fn, t, ody.QuantizedTensor(torch.from_numpy(w.data), w.kind, n * n),
                out=t)
    a = ody.Activation8(np.zeros((n, n), np.uint8), np.zeros((n, 1), np.uint8), n, n)
    refused(ody, L.ERR_ARG, "must not be or overlap an operand", ody.linear_wgrad8, x, a, out=x)
    lib, p = L.lib(), x.ctypes.data
    c, s = a.codes.ctypes.data, a.scales.ctypes.data
    assert lib.ody_fp4_linear(L.Q_NVFP4, p, 1.0, n, n, x.ctypes.data + 64, L.F32, 1, p, L.F32) == L.ERR_ARG
    assert lib.ody_linear_wgrad8(0, c, s, 1, n, p, L.F32, 1, 1.0, None, c, L.F32) == L.ERR_ARG
    assert lib.ody_linear_wgrad8(0, c, s, 1, n, p, L.F32, 1, 1.0, None, s, L.F32) == L.ERR_ARG
    for act8 in (lambda x, c, s: lib.ody_act8_save(0, x, L.F32, 1, n, c, s), lambda x, c, s: lib.ody_act8_load(0, c, s, 1, n, x, L.F32)):
        assert act8(p, p, s) == L.ERR_ARG and act8(p, c, p) == L.ERR_ARG and act8(p, c, c) == L.ERR_ARG
    # neither accumulation in place nor neighbouring buffers are (without a GPU they fail behind the checks)
    if not torch.cuda.is_available():
        acc = np.zeros((n, n), np.float32)
        refused(ody, L.ERR_CUDA, None, ody.linear_wgrad8, x[:, :16], a, add=acc[:16], out=acc[:16])
        refused(ody, L.ERR_CUDA, None, ody.fp4_linear, x[:16], w, out=x[16:])


def test_workspace_of_a_kind(ody):
    """Few rows of whole blocks take none, whatever the other kinds' blocks
    are; the query without a kind covers every kind."""
    from odyssey_b200 import _lib as L
    of, any_kind = L.lib().ody_linear_workspace_of, L.lib().ody_linear_workspace
    kinds = (L.Q_MXFP4, L.Q_NVFP4, L.Q_NVFP4_TENSOR, L.Q_MXFP4_OCP)
    for op, most in ((L.LINEAR_FORWARD, 32), (L.LINEAR_DGRAD, 16)):
        for dtype, parts in ((L.F32, 3), (L.F16, 2), (L.BF16, 1)):
            for rows in (1, most // parts, most // parts + 1, 200, 2048):
                for inn in (8192, 8176, 8168):
                    need = {k: of(op, k, rows, 8192, inn, dtype) for k in kinds}
                    assert any_kind(op, rows, 8192, inn, dtype) == max(need.values())
                    for k in kinds:
                        block = 32 if k in (L.Q_MXFP4, L.Q_MXFP4_OCP) else 16
                        few = rows * parts <= most and inn % block == 0
                        assert (need[k] == 0) == few, (op, dtype, rows, inn, k)
    for bad in ((3, 6, 1, 1, 1, 0), (0, 3, 1, 1, 1, 0), (1, 10, 1, 1, 1, 0), (0, 6, 0, 1, 1, 0), (0, 6, 1, 1, 1, 7)):
        assert of(*bad) == -1
    assert of(L.LINEAR_WGRAD, L.A8_E5M2, 8192, 4096, 4096, L.BF16) == any_kind(L.LINEAR_WGRAD, 8192, 4096, 4096, L.BF16) > 0


def test_weights_that_are_not_bytes_are_refused(ody):
    """As many elements as the weight has bytes, of another size, are not its
    bytes."""
    from odyssey_b200 import _lib as L
    import torch
    n = L.quant_bytes(L.Q_NVFP4, 8 * 16)
    x = np.ones((2, 16), np.float32)
    for dtype in (np.int16, np.float32, np.int64):
        w = ody.QuantizedTensor(np.zeros(n, dtype), L.Q_NVFP4, 8 * 16)
        refused(ody, L.ERR_DTYPE, "must be uint8", ody.fp4_linear, x, w)
        refused(ody, L.ERR_DTYPE, "must be uint8", ody.fp4_linear_dgrad, x[:, :8], w)
        t = ody.QuantizedTensor(torch.from_numpy(w.data), L.Q_NVFP4, 8 * 16)
        refused(ody, L.ERR_DTYPE, "must be uint8", ody.fp4_linear, torch.from_numpy(x), t)


def test_products_refuse_to_drop_a_gradient(ody):
    """The layer's gradients are calls of their own and no graph is recorded:
    a tensor that asks for one is turned away, unless gradients are off."""
    from odyssey_b200 import _lib as L
    import torch
    n = 32
    w = ody.QuantizedTensor(torch.zeros(L.quant_bytes(L.Q_NVFP4, n * n), dtype=torch.uint8), L.Q_NVFP4, n * n)
    a = ody.Activation8(torch.zeros(4, n, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 4, n)
    x, g = torch.ones(4, n), torch.ones(4, n, requires_grad=True)
    acc = torch.zeros(n, n, requires_grad=True)
    calls = [(ody.fp4_linear, (g, w), {}), (ody.fp4_linear, (g * 2, w), {}), (ody.fp4_linear, (x, w), {"out": g}),
             (ody.fp4_linear_dgrad, (g, w), {}), (ody.linear_wgrad8, (g, a), {}), (ody.linear_wgrad8, (x, a), {"add": acc}),
             (ody.linear_wgrad8, (x, a), {"out": acc})]
    for fn, args, kw in calls:
        refused(ody, L.ERR_ARG, "records no gradient", fn, *args, **kw)
    if not torch.cuda.is_available():  # with gradients off, and for data, the checks let them through
        for fn, args, kw in calls:
            with torch.no_grad():
                refused(ody, L.ERR_CUDA, None, fn, *args, **kw)
        refused(ody, L.ERR_CUDA, None, ody.fp4_linear, g.detach(), w)
        refused(ody, L.ERR_CUDA, None, ody.save_activation8, g)


def test_a_named_type_has_the_array_s_element_size(ody):
    """dtype= names the type of raw bits; it does not convert, and a type of
    another size would read past the array or half of it."""
    from odyssey_b200 import _lib as L
    w = weight(ody, 8, 16)
    f32, f16, u16 = np.ones((2, 16), np.float32), np.ones((2, 16), np.float16), np.ones((2, 16), np.uint16)
    for x, dtype in ((f32, "bfloat16"), (f32, "float16"), (f16, "float32"), (u16, "float32"), (f32, L.BF16), (f16.astype(float), "float32")):
        refused(ody, L.ERR_DTYPE, "elements of", ody.fp4_linear, x, w, dtype=dtype)
        refused(ody, L.ERR_DTYPE, "elements of", ody.save_activation8, x, dtype=dtype)
        refused(ody, L.ERR_DTYPE, "elements of", ody.quantize, x, L.Q_MXFP4, dtype=dtype)
        refused(ody, L.ERR_DTYPE, "elements of", ody.check_gradients_finite, x, dtype=dtype)
    for x, dtype in ((f32, "float64"), (f16, 7)):
        refused(ody, L.ERR_DTYPE, "unsupported dtype", ody.fp4_linear, x, w, dtype=dtype)
    for x, dtype in ((f32, "float32"), (f16, "float16"), (u16, "float16"), (u16, "bfloat16"), (u16.view(np.int16), "bfloat16")):
        assert L.dtype_code(x, dtype) == L.dtype_code(x, L.dtype_code(x, dtype))
