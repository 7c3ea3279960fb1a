"""Single tokens over the cache in 8 bits whose queries have features of very different size."""
from __future__ import annotations

import pytest
import torch

from test_gpu_kv8 import Rig

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("nh,nkv,d", [(8, 2, 128), (12, 1, 64)])
@pytest.mark.parametrize("power", [0, 16, 18, 20, 22, 24, 28])
def test_small_features_beside_a_large_one(power, nh, nkv, d, fmt):
    """One feature is 2^power times the others, and the keys are zero there: the scores are the others' products, which have all of
    their bits whatever stands beside them."""
    positions = [100, 191, 300]
    rig = Rig([p + 1 for p in positions], fmt=fmt, nh=nh, nkv=nkv, d=d, seed=power)
    for i, p in enumerate(positions):
        rig.k[i][:, :, 7] = 0
        rig.load(i, p)
    q = rig.rows(len(positions), nh, d)
    q[:, :, 7] = 2.0 ** power
    q, out = rig.decode(positions, q=q)
    for i, p in enumerate(positions):
        rig.check(i, q[i:i + 1], out[i:i + 1], [p])
