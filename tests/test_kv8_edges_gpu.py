"""Appending to the cache of 8-bit codes on a B200: sessions of a batch that add nothing."""
import numpy as np
import pytest

import clori_b200
from clori_b200 import abi
from tests.test_kv8_gpu import Cache, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", [abi.KV_E4M3, abi.KV_I8])
@pytest.mark.parametrize("held", [0.0, np.nan, 2.0 ** -140])
def test_a_session_without_new_rows_is_left_alone(backend, code, held):
    # slot 0 is idle (a length of its last session, no pages), slot 2 shares its last page, whose scales no append wrote
    rng = np.random.default_rng(71)
    heads, hd, page = 2, 64, 16
    cache = Cache(rng, 5, heads, page, hd, code)
    for which in range(2):
        cache.scales[which][3] = held
    device = cache.upload(backend)
    table = np.array([[-1, -1], [2, -1], [4, 3]], np.int32)
    x = clori_b200.bf16_bits_to_f32(clori_b200.f32_to_bf16_bits(rng.standard_normal((2, 3, 4, heads * hd)).astype(np.float32)))
    up = [backend.tensor("x", clori_b200.f32_to_bf16_bits(a)) for a in x]
    rc, _ = backend.kv8_append(up[0], up[1], *device, backend.tensor("t", table), kv_code=code, max_kv_tokens=27,
                               kv_tokens=backend.tensor("l", np.array([27, 5, 21], np.int32)),
                               new_tokens=backend.tensor("n", np.array([0, 4, 0], np.int32)))
    assert rc == 0
    for which in range(2):
        cache.append(which, table[1], 5, x[which, 1].reshape(4, heads, hd).astype(np.float64))
        assert np.array_equal(device[2 + which].read(), cache.scales[which], equal_nan=True)
        assert same(device[which].read(), cache.codes[which], code)
