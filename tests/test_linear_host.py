"""The quantised linear layer's refusals and host logic, without a GPU: every
case below is turned away before any device work."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def ody():
    from odyssey_b200.build import build
    build()
    import odyssey_b200
    odyssey_b200.lib()
    return odyssey_b200


def weight(ody, out, inn, kind=7):
    from odyssey_b200 import _lib as L
    return ody.QuantizedTensor(np.zeros(L.quant_bytes(kind, out * inn), np.uint8), kind, out * inn)


def refused(ody, code, match, fn, *args, **kw):
    with pytest.raises(ody.OdysseyError, match=match) as e:
        fn(*args, **kw)
    assert e.value.code == code


def test_product_refusals(ody):
    from odyssey_b200 import _lib as L
    w = weight(ody, 8, 16)
    x = np.ones((2, 16), np.float32)
    refused(ody, L.ERR_SHAPE, "has no rows of 15", ody.fp4_linear, x[:, :15], w)
    refused(ody, L.ERR_SHAPE, "does not have 9 rows", ody.fp4_linear_dgrad, np.ones((2, 9), np.float32), w)
    refused(ody, L.ERR_SHAPE, "is empty", ody.fp4_linear, x[:0], w)
    refused(ody, L.ERR_SHAPE, "is empty", ody.fp4_linear, x[:, :0], w)
    refused(ody, L.ERR_SHAPE, "is empty", ody.fp4_linear, np.float32(1.0), w)
    refused(ody, L.ERR_DTYPE, "unsupported dtype", ody.fp4_linear, x.astype(np.float64), w)
    refused(ody, L.ERR_DTYPE, "unsupported dtype", ody.fp4_linear, x, w, out_dtype="float64")
    refused(ody, L.ERR_ARG, "4-bit kinds", ody.fp4_linear, x, ody.QuantizedTensor(w.data, L.Q_FP8_E4M3, 128))
    refused(ody, L.ERR_ARG, "4-bit kinds", ody.fp4_linear, x, w.data)
    refused(ody, L.ERR_SHAPE, "bytes, expected", ody.fp4_linear, x, ody.QuantizedTensor(w.data[:-1], 7, 128))
    refused(ody, L.ERR_SHAPE, "out has shape", ody.fp4_linear, x, w, out=np.empty((2, 9), np.float32))
    refused(ody, L.ERR_DTYPE, "out must be float32", ody.fp4_linear, x, w, out=np.empty((2, 8), np.float16))
    refused(ody, L.ERR_ARG, "C-contiguous", ody.fp4_linear, x, w, out=np.empty((8, 2), np.float32).T)


def test_activation_refusals(ody):
    from odyssey_b200 import _lib as L
    x = np.ones((3, 40), np.float32)
    refused(ody, L.ERR_ARG, "unknown 8-bit activation format", ody.save_activation8, x, "e3m4")
    refused(ody, L.ERR_SHAPE, "is empty", ody.save_activation8, x[:0])
    codes, scales = np.zeros((3, 64), np.uint8), np.zeros((3, 2), np.uint8)
    ok = ody.Activation8(codes, scales, 3, 40)
    dy = np.ones((3, 8), np.float32)
    A = ody.Activation8
    refused(ody, L.ERR_SHAPE, "do not have the bytes", ody.load_activation8, A(codes[:, :40], scales, 3, 40))
    refused(ody, L.ERR_SHAPE, "do not have the bytes", ody.load_activation8, A(codes, scales[:, :1], 3, 40))
    refused(ody, L.ERR_DTYPE, "must be uint8", ody.load_activation8, A(codes.astype(np.int16), scales, 3, 40))
    refused(ody, L.ERR_ARG, "unknown 8-bit", ody.load_activation8, A(codes, scales, 3, 40, "fp8"))
    refused(ody, L.ERR_SHAPE, "empty activation", ody.load_activation8, A(codes[:0], scales[:0], 0, 40))
    refused(ody, L.ERR_SHAPE, "dy has 2 rows", ody.linear_wgrad8, dy[:2], ok)
    refused(ody, L.ERR_SHAPE, "add has shape", ody.linear_wgrad8, dy, ok, add=np.ones((8, 41), np.float32))
    refused(ody, L.ERR_DTYPE, "add must be float16", ody.linear_wgrad8, dy, ok, add=np.ones((8, 40), np.float32),
            out_dtype="float16")
    refused(ody, L.ERR_SHAPE, "out has shape", ody.linear_wgrad8, dy, ok, out=np.ones((40, 8), np.float32))


def test_c_entry_refusals(ody):
    """The C entries check for themselves (nothing here reaches a launch)."""
    from odyssey_b200 import _lib as L
    lib = L.lib()
    b = np.zeros(4096, np.uint8)
    p = b.ctypes.data

    def lin(kind=7, q=p, out=8, inn=16, x=p, xd=0, rows=2, ld=16, y=p, yd=0, ldy=8):
        return lib.ody_fp4_linear_on_stream(kind, q, None, 1.0, out, inn, x, xd, rows, ld, y, yd, ldy, None, 0, None)

    assert lin(kind=3) == L.ERR_ARG and lin(kind=0) == L.ERR_ARG and lin(kind=10) == L.ERR_ARG
    assert lin(xd=3) == L.ERR_DTYPE and lin(yd=-1) == L.ERR_DTYPE
    assert lin(rows=0) == L.ERR_SHAPE and lin(out=-1) == L.ERR_SHAPE and lin(inn=0) == L.ERR_SHAPE
    assert lin(rows=2 ** 31) == L.ERR_SHAPE
    assert lin(ld=15) == L.ERR_SHAPE and lin(ldy=7) == L.ERR_SHAPE and lin(ld=2 ** 60) == L.ERR_SHAPE
    assert lin(q=None) == L.ERR_ARG and lin(x=None) == L.ERR_ARG and lin(y=None) == L.ERR_ARG
    assert lin() == L.ERR_ARG  # host memory at a stream entry
    assert lib.ody_act8_save_on_stream(2, p, 0, 1, 32, 32, p, p, None) == L.ERR_ARG
    assert lib.ody_act8_save_on_stream(0, p, 5, 1, 32, 32, p, p, None) == L.ERR_DTYPE
    assert lib.ody_act8_save_on_stream(0, p, 0, 0, 32, 32, p, p, None) == L.ERR_SHAPE
    assert lib.ody_act8_save_on_stream(0, p, 0, 1, 32, 31, p, p, None) == L.ERR_SHAPE
    assert lib.ody_act8_load_on_stream(0, None, p, 1, 32, p, 0, 32, None) == L.ERR_ARG
    assert lib.ody_act8_load_on_stream(0, p, p, 1, 32, p, 0, 32, None) == L.ERR_ARG
    assert lib.ody_linear_wgrad8(4, p, p, 1, 32, p, 0, 8, 1.0, None, p, 0) == L.ERR_ARG
    assert lib.ody_linear_wgrad8(0, p, None, 1, 32, p, 0, 8, 1.0, None, p, 0) == L.ERR_ARG
    assert lib.ody_linear_wgrad8(0, p, p, 1, 32, p, 0, 0, 1.0, None, p, 0) == L.ERR_SHAPE
    assert [lib.ody_act8_groups(c) for c in (-1, 0, 1, 32, 33)] == [0, 0, 1, 1, 2]


def test_workspace_query(ody):
    from odyssey_b200 import _lib as L
    ws = L.lib().ody_linear_workspace
    for bad in ((3, 1, 1, 1, 0), (-1, 1, 1, 1, 0), (0, 0, 1, 1, 0), (0, 1, -5, 1, 0), (0, 1, 1, 2 ** 40, 0), (0, 1, 1, 1, 7)):
        assert ws(*bad) == -1
    for op in range(3):
        for dt in range(3):
            assert ws(op, 1, 1, 1, dt) >= 0 and ws(op, 4096, 4096, 4096, dt) >= 0


def test_no_gpu_fails_loudly(ody):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    from odyssey_b200 import _lib as L
    refused(ody, L.ERR_CUDA, "", ody.fp4_linear, np.ones((2, 16), np.float32), weight(ody, 8, 16))
    refused(ody, L.ERR_CUDA, "", ody.save_activation8, np.ones((2, 16), np.float32))


def test_reference_statements():
    """The float64 statements the GPU tests use, on hand-worked values."""
    import linear_ref as R
    assert list(R.e4m3([0, 1, 8, 56, 0x7E, 0x80 + 56])) == [0, 2.0 ** -9, 2.0 ** -6, 1.0, 448.0, -1.0]
    assert list(R.e5m2([0, 1, 4, 60, 0x7B, 0x7C])) == [0, 2.0 ** -16, 2.0 ** -14, 1.0, 57344.0, np.inf]
    q = np.zeros(17, np.uint8)
    q[0], q[1], q[16] = 0x2F, 0x91, 128  # elements 1.0, -6.0, -(0 or 0.5), 0 or 0.5; scale 2
    assert list(R.weight(R.MXFP4, q, 1, 4)[0]) == [2.0, -12.0, 0.0, 0.0]
    assert list(R.weight(R.MXFP4_OCP, q, 1, 4)[0]) == [2.0, -12.0, -1.0, 1.0]
    v, p = R.encode8(np.array([[448.0, 1.0, 17.0, 19.0, 0.001]]), "e4m3")
    assert p[0, 0] == 0 and list(v[0]) == [448.0, 1.0, 16.0, 20.0, 2.0 ** -9]
    v, p = R.encode8(np.array([[449.0, 1.0]]), "e4m3")
    assert p[0, 0] == 1 and list(v[0]) == [448.0, 1.0]
    v, p = R.encode8(np.array([[0.0, np.inf, np.nan, 3.0]]), "e5m2")
    assert v[0, 1] == np.inf and np.isnan(v[0, 2]) and v[0, 3] == 3.0 and p[0, 0] == -14
    v, _ = R.encode8(np.array([[np.inf, 3.0]]), "e4m3")
    assert np.isnan(v[0, 0]) and v[0, 1] == 3.0
