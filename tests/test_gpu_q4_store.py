"""The 4-bit cache's write and read-back next to the format's limit and where values are rounded: stored bytes
and read values are exact against the 64-bit oracle."""
import numpy as np
import pytest
import torch

from oracle import q4 as O
from test_gpu_q4 import DT, GEOMETRIES, _lay, _np

pytestmark = pytest.mark.gpu


def _bytes(lay, k, v, bs=16):
    """The cache that holds token i in slot i, by the oracle."""
    want = np.zeros(tuple(lay.cache_shape(-(-len(k) // bs), bs)), np.uint8)
    kq, vq = O.quantise(_np(k), lay.group), O.quantise(_np(v), lay.group)
    for i in range(len(k)):
        for h in range(lay.H):
            O.put(want, i, h, bs, [a[i, h] for a in kq], [a[i, h] for a in vq])
    return want


@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_values_next_to_the_limit(d, g, dtype):
    """Groups that lie within a few hundred of +-57344 with values beyond it: the minimum is then rounded as far as
    the limit itself, and a code is that of the clamped value."""
    from vllm_ttkv import ops
    lay, n = _lay(2, d, g), 48
    rng = np.random.default_rng(d + g)
    x = 57344.0 - rng.uniform(0, 1, (2, n, 2, d)) * 10.0 ** rng.uniform(-2, 4, (2, n, 2, 1))
    x[:, ::3, :, ::5] = 57344.0 + 10.0 ** rng.uniform(-1, 4, x[:, ::3, :, ::5].shape)
    x[:, 1::3] = np.where(rng.uniform(size=x[:, 1::3].shape) < 0.2, 60000.0, x[:, 1::3])
    x[0, 0, :, :] = 57340.0                              # the limit's code is 0, not 15
    x[0, 0, :, 1::32] = 60000.0
    x[:, ::2] *= -1
    x[0, 0] *= -1
    k, v = (torch.from_numpy(a).to(DT[dtype]).cuda() for a in x)
    cache = lay.new_cache(n // 16, 16)
    ops.reset_status()
    ops.q4_write_paged(lay, cache, torch.arange(n, device="cuda"), k, v)
    ops.check_status()
    want = _bytes(lay, k, v)
    got = cache.cpu().numpy()
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
