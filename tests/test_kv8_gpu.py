"""The cache of 8-bit codes on a B200: appended codes and scales are equal to the definition in float64, code by code."""
import numpy as np
import pytest

import clori_b200
from clori_b200 import abi
from tests.scored_cases import decode, encode, power_scale

pytestmark = pytest.mark.gpu
E4M3, I8 = abi.KV_E4M3, abi.KV_I8


class Cache:
    """Host twin of a pool of codes: what every append is required to leave behind."""

    def __init__(self, rng, pages, heads, page, hd, code):
        self.code, self.page = code, page
        self.codes = [rng.integers(0, 256, (pages, heads, page, hd)).astype(np.uint8) for _ in range(2)]
        self.scales = [np.exp2(rng.integers(-20, 20, (pages, heads))).astype(np.float32) for _ in range(2)]

    def append(self, which, table, present, rows):
        """rows [n, heads, hd] float64 behind `present` rows of one session."""
        codes, scales, page = self.codes[which], self.scales[which], self.page
        n = rows.shape[0]
        for j in range(present // page, -(-(present + n) // page)):
            block, lo, hi = table[j], max(present, j * page), min(present + n, (j + 1) * page)
            kept = lo - j * page
            for h in range(rows.shape[1]):
                new = rows[lo - present:hi - present, h]
                new = np.where(np.isfinite(new), new, 0.0)
                s = power_scale(np.abs(new).max(), self.code)
                if kept:
                    held = float(scales[block, h])
                    s = max(s, held)
                    if s > held:
                        old = decode(codes[block, h, :kept], self.code)
                        again = encode(np.nan_to_num(old) * (held / s), self.code)
                        codes[block, h, :kept] = np.where(np.isnan(old), codes[block, h, :kept], again)
                codes[block, h, kept:hi - j * page] = encode(new / s, self.code)
                scales[block, h] = s

    def upload(self, backend):
        shape = self.codes[0].shape
        return [backend.tensor("c", c.view(np.int8)) for c in self.codes] + [backend.tensor("s", s) for s in self.scales]


def tables(rng, lengths, page, spare=2):
    need = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    table = np.full((len(need), max(1, max(need))), -1, np.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    return table, len(order)


def same(got, want, code):
    """Codes stand for the same values: e4m3 has two zeros and two NaN codes."""
    return np.array_equal(decode(got.view(np.uint8), code), decode(want, code), equal_nan=True)


CASES = [
    # present rows, new rows, heads, hd, page
    ([0], [1], 1, 128, 64),
    ([5, 0, 63, 64, 100], [1, 1, 1, 1, 1], 8, 128, 64),
    ([37, 37], [200, 130], 3, 128, 64),
    ([0, 15, 16, 31], [17, 1, 40, 2], 2, 64, 16),
    ([10, 3], [0, 300], 2, 256, 128),
    ([9], [25], 5, 16, 7),
    ([250, 1], [300, 600], 1, 48, 256),
    ([127, 0], [2, 31], 2, 128, 32),
]


@pytest.mark.parametrize("code", [E4M3, I8])
@pytest.mark.parametrize("dtype", [abi.DTYPE_BF16, abi.DTYPE_F32])
@pytest.mark.parametrize("present,fresh,heads,hd,page", CASES)
def test_append_equals_the_definition(backend, code, dtype, present, fresh, heads, hd, page):
    rng = np.random.default_rng(3 * page + heads)
    tokens, S = max(fresh), len(present)
    table, pages = tables(rng, [a + tokens for a in present], page)
    cache = Cache(rng, pages, heads, page, hd, code)
    device = cache.upload(backend)
    lens, new = np.array(present, np.int32), np.array(fresh, np.int32)
    for step in range(3):                    # louder each time: held scales have to grow, then stay
        x = [(rng.standard_normal((S, tokens, heads, hd)) * 10.0 ** ((0, 3, -2)[step])).astype(np.float32) for _ in range(2)]
        for a in x:
            a[:, :, :, 0] *= 7.0
            if step == 0:
                a[0, :, 0] = 0.0             # a page of zeros takes the smallest scale
        bits = [clori_b200.f32_to_bf16_bits(a) for a in x]
        values = [clori_b200.bf16_bits_to_f32(b) for b in bits] if dtype == abi.DTYPE_BF16 else x
        up = [backend.tensor("x", (b if dtype == abi.DTYPE_BF16 else a).reshape(S, tokens, heads * hd)) for a, b in zip(x, bits)]
        rc, facts = backend.kv8_append(up[0], up[1], *device, backend.tensor("t", table), kv_code=code,
                                       max_kv_tokens=max(present), kv_tokens=backend.tensor("l", lens),
                                       new_tokens=backend.tensor("n", new))
        assert rc == 0 and facts.kernel_launches == 1
        for b in range(S):
            for which in range(2):
                if fresh[b]:
                    cache.append(which, table[b], present[b], values[which][b, :fresh[b]].astype(np.float64))
        for which in range(2):
            assert np.array_equal(device[2 + which].read(), cache.scales[which])
            assert same(device[which].read(), cache.codes[which], code)


@pytest.mark.parametrize("code", [E4M3, I8])
def test_rows_one_by_one_equal_what_their_scales_allow(backend, code):
    # a page filled token by token: the final scale is that of the loudest row, and every value is within the half
    # steps that it was rounded by: once when stored and once for each growth of the scale behind it
    rng = np.random.default_rng(9)
    heads, hd, page, n = 2, 128, 64, 64
    cache = Cache(rng, 2, heads, page, hd, code)
    device = cache.upload(backend)
    table = np.array([[1]], np.int32)
    x = clori_b200.bf16_bits_to_f32(clori_b200.f32_to_bf16_bits((rng.standard_normal((2, n, heads, hd)) * np.exp(
        rng.standard_normal((2, n, heads, 1)))).astype(np.float32)))
    t = backend.tensor("t", table)
    for i in range(n):
        up = [backend.tensor("x", clori_b200.f32_to_bf16_bits(x[w, i].reshape(1, 1, heads * hd))) for w in range(2)]
        backend.kv8_append(up[0], up[1], *device, t, kv_code=code, max_kv_tokens=i)
        for w in range(2):
            cache.append(w, table[0], i, x[w, i:i + 1].astype(np.float64))
    for w in range(2):
        scales = device[2 + w].read()[1].astype(np.float64)
        assert scales.tolist() == [power_scale(np.abs(x[w][:, h]).max(), code) for h in range(heads)]
        assert same(device[w].read(), cache.codes[w], code)


def test_strided_and_misaligned_rows(backend):
    rng = np.random.default_rng(21)
    heads, hd, page, tokens = 2, 64, 16, 20
    for dtype, stride, shift in ((abi.DTYPE_BF16, 2 * heads * hd, 0), (abi.DTYPE_BF16, heads * hd + 3, 0),
                                 (abi.DTYPE_F32, 2 * heads * hd + 1, 0)):
        cache = Cache(rng, 4, heads, page, hd, E4M3)
        device = cache.upload(backend)
        x = [rng.standard_normal((1, tokens, stride)).astype(np.float32) for _ in range(2)]
        if dtype == abi.DTYPE_BF16:
            x = [clori_b200.bf16_bits_to_f32(clori_b200.f32_to_bf16_bits(a)) for a in x]
        up = [backend.tensor("x", clori_b200.f32_to_bf16_bits(a) if dtype == abi.DTYPE_BF16 else a) for a in x]
        table = np.array([[3, 0]], np.int32)
        backend.kv8_append(up[0], up[1], *device, backend.tensor("t", table), kv_code=E4M3, max_kv_tokens=0,
                           token_stride=stride)
        for w in range(2):
            cache.append(w, table[0], 0, x[w][0, :, :heads * hd].reshape(tokens, heads, hd).astype(np.float64))
            assert same(device[w].read(), cache.codes[w], E4M3) and np.array_equal(device[2 + w].read(), cache.scales[w])


def test_lanes_that_are_not_finite_are_zero_and_reported(backend):
    rng = np.random.default_rng(1)
    for code in (E4M3, I8):
        cache = Cache(rng, 1, 1, 16, 32, code)
        device = cache.upload(backend)
        x = rng.standard_normal((1, 4, 32)).astype(np.float32)
        x[0, 1, 3], x[0, 2, 5], x[0, 3, 31] = np.nan, np.inf, -np.inf
        values = rng.standard_normal((1, 4, 32)).astype(np.float32)
        up = [backend.tensor("x", x), backend.tensor("x", values)]
        rc, _ = backend.kv8_append(up[0], up[1], *device, backend.tensor("t", np.zeros((1, 1), np.int32)), kv_code=code,
                                   max_kv_tokens=0, check=False)
        assert rc == abi.YVEX_ERR_FORMAT
        table = np.zeros(1, np.int32)
        cache.append(0, table, 0, x.reshape(4, 1, 32).astype(np.float64))
        cache.append(1, table, 0, values.reshape(4, 1, 32).astype(np.float64))
        for w in range(2):
            device[w].struct.is_written = device[2 + w].struct.is_written = 1
            assert same(device[w].read(), cache.codes[w], code) and np.array_equal(device[2 + w].read(), cache.scales[w])


def test_bad_tables_and_lengths_write_nothing(backend):
    rng = np.random.default_rng(2)
    heads, hd, page = 2, 32, 16
    x = backend.tensor("x", rng.standard_normal((2, 3, heads * hd)).astype(np.float32))
    for lens, new, table in (([0, 0], [3, 3], [[0, -1], [9, 1]]), ([0, 31], [3, 3], [[0, 1], [2, 3]]),
                             ([0, -4], [3, 3], [[0, 1], [2, 3]]), ([0, 0], [3, 9], [[0, 1], [2, 3]])):
        cache = Cache(rng, 4, heads, page, hd, I8)
        device = cache.upload(backend)
        rc, _ = backend.kv8_append(x, x, *device, backend.tensor("t", np.array(table, np.int32)), kv_code=I8, max_kv_tokens=16,
                                   kv_tokens=backend.tensor("l", np.array(lens, np.int32)),
                                   new_tokens=backend.tensor("n", np.array(new, np.int32)), check=False)
        assert rc == abi.YVEX_ERR_FORMAT
        values = x.read().reshape(2, 3, heads, hd).astype(np.float64)
        for w in range(2):                   # the first session is sound, the second is skipped
            cache.append(w, np.array(table[0]), 0, values[0])
            assert same(device[w].read(), cache.codes[w], I8) and np.array_equal(device[2 + w].read(), cache.scales[w])


def test_operator_refusals(backend):
    z = lambda shape, t=np.int8: backend.tensor("z", np.zeros(shape, t))
    heads, hd, page = 2, 64, 16
    x, codes, scales, table = z((1, 4, heads * hd), np.float32), z((3, heads, page, hd)), z((3, heads), np.float32), z((1, 2), np.int32)

    def call(key=x, code=E4M3, k_codes=codes, k_scales=scales, **fields):
        return backend.kv8_append(key, x, k_codes, codes, k_scales, scales, table, kv_code=code, max_kv_tokens=0,
                                  check=False, **fields)[0]
    assert call() == 0
    assert call(code=0) == abi.YVEX_ERR_UNSUPPORTED
    assert call(key=z((1, 4, heads * hd), np.uint16)) == abi.YVEX_ERR_UNSUPPORTED      # K and V of two types
    assert call(token_count=40) == abi.YVEX_ERR_BOUNDS
    assert call(token_count=20) == abi.YVEX_ERR_FORMAT                                 # more rows than the tensors hold
    assert call(k_codes=z((3, heads, page, hd), np.float32)) == abi.YVEX_ERR_FORMAT
    assert call(k_scales=z((3, heads))) == abi.YVEX_ERR_FORMAT
    assert call(session_count=0) == abi.YVEX_ERR_INVALID_ARG
    assert call(token_stride=heads * hd - 1) == abi.YVEX_ERR_INVALID_ARG
