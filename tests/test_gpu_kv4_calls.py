"""Calls of the 4-bit KV cache's operators in the forms that programs make of them: all layers at
once, on other streams than the tensors' own, inside captures, through the model and the batcher.
Oracle and tolerances: tests/test_gpu_kv4.py."""
import numpy as np
import pytest
import torch

from oracle import kv4 as OK
from tests.test_gpu_kv4 import DT, dev, random_pool, rounded, tables_for

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv4(cuda_device):
    from tiny_infra_b200 import _native, kv4
    _native.device_status()
    yield kv4
    assert _native.device_status() == 0


@pytest.mark.parametrize("dtn", ["bf16", "fp16"])
@pytest.mark.parametrize("d,kvh,layers", [(64, 2, 3), (128, 1, 2)])
def test_evict_all_layers_and_read_them_back(kv4, dtn, d, kvh, layers):
    """The survivors of every layer, read back in one call from the pool that evict took: block
    ids count through the layers.  Exact."""
    rng = np.random.default_rng(d + layers)
    lens, keep, recent, dt = np.array([70, 16, 0, 33], np.int32), 32, 5, DT[dtn]
    new = np.minimum(lens, keep)
    tables, nb = tables_for(rng, lens)
    pool = np.stack([random_pool(rng, nb, kvh, d) for _ in range(layers)])
    w = rng.random((layers, nb, kvh, 16)).astype(np.float32)
    dp, dw = dev(pool), dev(w)
    kv4.evict(dp, dw, dev(tables), dev(lens), keep, recent)
    OK.evict(pool, w, tables, lens, keep, recent)
    most = keep // 16
    src = np.full((layers, len(lens), most), -1, np.int32)
    dst = src.copy()
    for la in range(layers):
        for i, n in enumerate(new):
            k = -(-int(n) // 16)
            src[la, i, :k] = la * nb + tables[i, :k]
            dst[la, i, :k] = (la * len(lens) + i) * most + np.arange(k)
    ko = torch.full((layers * len(lens) * most, kvh, 16, d), 9.0, dtype=dt, device="cuda")
    vo = ko.clone()
    kv4.dequantize(dp, dev(src.reshape(-1, most)), dev(np.tile(new, layers)),
                   dev(dst.reshape(-1, most)), ko, vo)
    for g, which in ((ko, 0), (vo, 1)):
        want = np.full(g.shape, 9.0)
        for la in range(layers):
            vals = OK.untile(pool[la])[which]
            for i, n in enumerate(new):
                for j in range(-(-int(n) // 16)):
                    x = vals[tables[i, j]].copy()
                    x[:, max(0, int(n) - 16 * j):] = 0
                    want[dst[la, i, j]] = x
        np.testing.assert_array_equal(g.double().cpu().numpy(), rounded(want, dt))
