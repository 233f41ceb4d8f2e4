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
