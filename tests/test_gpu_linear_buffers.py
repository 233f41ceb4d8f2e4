"""The quantised linear layer's buffers on the GPU: strided, shared and
pitched ones."""
import numpy as np
import pytest
import torch

import linear_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ody():
    import odyssey_b200
    odyssey_b200.lib()
    return odyssey_b200


def test_strided_host_weight(ody):
    """Every other byte of a buffer as the weight, in numpy and in torch."""
    rng = np.random.default_rng(1)
    out, inn = 1024, 1024
    q = R.random_weight(rng, R.NVFP4, out, inn)
    wide = rng.integers(0, 256, 2 * q.size, dtype=np.uint8)
    wide[::2] = q
    x = rng.standard_normal((3, 1024)).astype(np.float32)
    for fn in (ody.fp4_linear, ody.fp4_linear_dgrad):
        want = fn(x, ody.QuantizedTensor(q, R.NVFP4, out * inn))
        assert np.array_equal(fn(x, ody.QuantizedTensor(wide[::2], R.NVFP4, out * inn)), want)
        strided = ody.QuantizedTensor(torch.from_numpy(wide)[::2], R.NVFP4, out * inn)
        assert np.array_equal(fn(torch.from_numpy(x), strided).numpy(), want)


def test_host_results_over_their_operands(ody):
    """A host call of the stateless operations whose result takes an operand's
    place gives the result, not the operand."""
    from odyssey_b200 import _lib as L
    lib = L.lib()
    rng = np.random.default_rng(2)
    g, p, m, v = (rng.standard_normal(1000).astype(np.float32) for _ in range(4))
    v = np.abs(v)
    apart, over = np.empty_like(g), g.copy()
    L.check(lib.ody_unscale(g.ctypes.data, L.F32, 1000, 3.0, apart.ctypes.data))
    L.check(lib.ody_unscale(over.ctypes.data, L.F32, 1000, 3.0, over.ctypes.data))
    assert np.array_equal(over, apart) and not np.array_equal(over, g)
    want = ody.adamw_step(p, g, m, v, 1, 1e-3)
    args = [a.ctypes.data for a in (p, g, m, v)]
    L.check(lib.ody_adamw_step(*args, 1000, 1, 1e-3, 0.9, 0.999, 1e-8, 0.01, args[0], args[2], args[3]))
    for got, w in zip((p, m, v), want):
        assert np.array_equal(got, w)
