"""Scored attention on a B200 at the edges of what it accepts: gaps between the tokens that rows see, values far apart,
scores and caps far outside the usual range, positions far behind the cache, memory that follows what a call sees."""
import ctypes as C

import numpy as np
import pytest

import clori_b200
from clori_b200 import abi
from tests.scored_cases import WEIGHTS, Case, attention, tolerance

pytestmark = pytest.mark.gpu
E4M3, I8, PLAIN = abi.KV_E4M3, abi.KV_I8, abi.KV_PLAIN
F32, BF16 = abi.DTYPE_F32, abi.DTYPE_BF16


def runs(sessions, rows_runs):
    """row_first / row_end, the same for every session."""
    first, end = zip(*rows_runs)
    return np.tile(np.array(first), (sessions, 1)), np.tile(np.array(end), (sessions, 1))


@pytest.mark.parametrize("cache,page", [(E4M3, 16), (I8, 64), (E4M3, 128)])
@pytest.mark.parametrize("value", [np.nan, np.inf, 1e10])
@pytest.mark.parametrize("rows,path", [(1, "decode_codes"), (4, "decode_codes"), (33, "prompt"), (4, "general")])
@pytest.mark.parametrize("chunk", [None, 128, 1280])
def test_scales_of_pages_that_no_row_sees(backend, cache, page, value, rows, path, chunk):
    # two documents with padding of several pages between them; the padding's pages and scales were never written
    spans = ([(0, 200), (0, 129), (640, 1150), (700, 897)] * 9)[:rows]
    if rows == 1:
        spans = [(300, 301)]
    c = Case(41, [1200, 900], rows, 8, 2, 128, cache=cache, page=page, ranges=runs(2, spans))
    for b in range(2):
        for j in range(-(-int(c.lengths[b]) // page)):
            if not c.seen[b, j * page:(j + 1) * page].any():
                for x in ("k_scales", "v_scales"):
                    c.arrays[x][c.table[b, j]] = value
    c.check(backend, path, force_general=path == "general", chunk=chunk)


def lonely_nan(c, b, token):
    """The key of one token becomes NaN; where codes have none, by the scale of its page."""
    where = c._slot(b, token)
    if c.cache == I8:
        c.arrays["k_scales"][where[0]] = np.nan
    elif c.cache:
        c.arrays["k"][where] = 0x7f
    else:
        c.arrays["k"][where] = np.nan


NAN_CACHES = [dict(), dict(page=64), dict(cache=E4M3, page=64), dict(cache=I8, page=64)]


@pytest.mark.parametrize("fields", NAN_CACHES)
@pytest.mark.parametrize("sessions,heads", [(1, 4), (300, 8)])      # a block for each item of the fold, a warp for each
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_a_nan_that_fills_its_split_is_reported(backend, fields, sessions, heads, cap):
    # the newest token alone in its split of 64
    lengths = [321] + [65] * (sessions - 1)
    c = Case(42, lengths, 1, heads, 2, 128, garbage=False, cap=cap, **fields)
    lonely_nan(c, 0, 320)
    got, status = c.launch(backend, c.plan(backend, c.problem(backend), 64))
    assert status == 1 and np.isnan(got[0]).all() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("fields", NAN_CACHES)
@pytest.mark.parametrize("sessions,heads", [(1, 4), (300, 8)])
def test_a_query_of_nan_is_reported(backend, fields, sessions, heads):
    c = Case(43, [321] + [65] * (sessions - 1), 1, heads, 2, 128, garbage=False, **fields)
    c.q[0, 0, 1, 77] = np.nan
    got, status = c.launch(backend, c.plan(backend, c.problem(backend), 64))
    assert status == 1 and np.isnan(got[0, 0, 1]).all() and np.isfinite(got[0, 0, 0]).all() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("sessions,heads", [(1, 4), (300, 8)])
@pytest.mark.parametrize("rows,general", [(1, False), (1, True), (40, False)])
def test_a_nan_in_a_split_of_no_weight_is_reported(backend, sessions, heads, rows, general):
    # the split's finite logits lie hundreds below those of the other splits
    if rows > 1:
        sessions = min(sessions, 20)
    c = Case(44, [322] + [322] * (sessions - 1), rows, heads, 2, 128, garbage=False, causal=False)
    c.q[:] = 1.0
    c.arrays["k"][:] = 20.0
    c.arrays["k"][0, 257:] = -20.0
    c.arrays["k"][0, 256] = np.nan
    got, status = c.launch(backend, c.plan(backend, c.problem(backend, general), 128 if rows > 1 else 64))
    assert status == 1 and np.isnan(got[0]).all() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("apart", [30, 40, 80])
@pytest.mark.parametrize("chunk", [None, 128, 384])
def test_scales_of_values_far_apart(backend, cache, apart, chunk):
    # a document for each tile of 64 tokens, their values 2^30 and more apart, up and down; the last rows see two of them
    spans = [(64 * i + 3, 64 * i + 60) for i in range(6)] + [(130, 250), (0, 384)]
    c = Case(45, [384], 8, 2, 2, 128, cache=cache, page=16, ranges=runs(1, spans))
    power = np.array([0, apart, 0, -apart, apart, -apart])
    for j in range(24):
        c.arrays["v_scales"][c.table[0, j]] *= 2.0 ** power[j // 4]
    c.values["v"][0] *= 2.0 ** np.repeat(power, 64)[:, None, None]
    c.check(backend, "decode_codes", chunk=chunk)


@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("chunk", [None, 128, 384])
def test_large_values_of_small_weight(backend, cache, chunk):
    # one tile in three holds values 2^60 times the others' at a weight of 2^-65: both carry the result
    c = Case(46, [384], 1, 2, 2, 128, cache=cache, page=16, garbage=False)
    c.q[:] = 1.0
    one = 0x38 if cache == E4M3 else 1
    c.arrays["k"][:] = one
    c.values["k"][:] = 1.0
    c.arrays["k_scales"][:] = 4.0
    c.values["k"] *= 4.0
    for j in range(24):
        if j // 4 % 3 == 1:
            block = c.table[0, j]
            c.arrays["k"][block] = 0xb8 if cache == E4M3 else 0xff
            c.arrays["v_scales"][block] *= 2.0 ** 60
            c.values["k"][0, 16 * j:16 * j + 16] *= -1.0
            c.values["v"][0, 16 * j:16 * j + 16] *= 2.0 ** 60
    c.q *= 0.5                                  # logits of +-22.6: weights 2^-65 apart
    c.check(backend, "decode_codes", chunk=chunk)


# A logit under a cap may be off by this much of itself: tanh from its exponential or from a polynomial of its own, relative
# to the result; the prompt kernel's polynomial for small arguments starts with 0.99999061 x.
CAP_RELATIVE = {"general": 2.0 ** -21, "decode_bf16": 2.0 ** -20, "decode_codes": 2.0 ** -20, "prompt": 2.0 ** -16}


def check_cap(c, backend, path):
    got, status = c.launch(backend, c.plan(backend, c.problem(backend, path == "general")))
    assert status == 0
    for b in range(len(c.lengths)):
        want, spread, size = attention(c.q[b].astype(np.float64), c.values["k"][b], c.values["v"][b], c.position[b], c.first[b],
                                       c.end[b], float(np.float32(1 / np.sqrt(128))), float(np.float32(c.cap)))
        visible = np.broadcast_to((c.end - c.first)[b][:, None].astype(np.float64), size.shape)
        # size bounds |z|; tolerance() takes 2^-20 of its `cap`
        allowed = tolerance(want, spread, size, visible, 128, WEIGHTS[path], 2.0 ** -24, size * CAP_RELATIVE[path] * 2.0 ** 20)
        assert np.all(np.abs(got[b] - want) <= allowed), float((np.abs(got[b] - want) / allowed).max())


CAPPED = [(2, "decode_bf16", {}), (70, "prompt", dict(ranges=True)), (2, "decode_codes", dict(cache=E4M3, page=16)), (1, "decode_codes", dict(cache=I8, page=64)),
          (70, "prompt", {}), (3, "general", {})]


@pytest.mark.parametrize("cap", [63.0, 65.0, 1e3, 2047.0, 2049.0, 1e5, 1e6, 1e7, 1e30, 1e38])
@pytest.mark.parametrize("rows,path,fields", CAPPED)
def test_moderate_logits_under_a_large_cap(backend, cap, rows, path, fields):
    if fields.get("ranges"):
        fields = dict(ranges=runs(2, [(3 * i, 3 * i + 60) for i in range(rows)]))
    check_cap(Case(47, [300, 280], rows, 4, 2, 128, cap=cap, q_scale=3.0, **fields), backend, path)


@pytest.mark.parametrize("cap", [1e3, 3e3, 1e5])
@pytest.mark.parametrize("rows,path,fields", CAPPED)
def test_one_loud_row_beside_moderate_ones_under_a_large_cap(backend, cap, rows, path, fields):
    # the loud row's logits leave the part of the curve where tanh x is nearly x, its neighbours' do not
    if fields.get("ranges"):
        fields = dict(ranges=runs(2, [(3 * i, 3 * i + 60) for i in range(rows)]))
    c = Case(48, [300, 280], rows, 4, 2, 128, cap=cap, q_scale=2.0, **fields)
    c.q[:, 0, 1] *= 2.0 ** np.ceil(np.log2(cap))
    check_cap(c, backend, path)


@pytest.mark.parametrize("scale,q_scale,k_scale", [(1e-30, 1.0, 1.0), (1e-25, 1e3, 1e3), (1e-13, 1e6, 1e6), (1e30, 2.0 ** -50, 2.0 ** -49),
                                                  (2e12, 2.0 ** -20, 2.0 ** -20)])
@pytest.mark.parametrize("rows,fields", [(70, {}), (70, dict(slopes=True)), (70, dict(ranges=True)), (2, {}), (70, dict(cap=20.0)),
                                         (40, dict(cache=E4M3, page=64))])
def test_extreme_scales(backend, scale, q_scale, k_scale, rows, fields):
    fields = dict(fields)
    if fields.get("ranges"):
        fields["ranges"] = runs(2, [(3 * i, 3 * i + 60) for i in range(rows)])
    c = Case(49, [300, 290], rows, 4, 2, 128, q_scale=q_scale, k_scale=k_scale, **fields)
    p = c.problem(backend)
    p.scale = scale
    got, status = c.launch(backend, c.plan(backend, p))
    assert status == 0
    slopes = None if c.slope is None else c.slope.astype(np.float64)
    for b in range(2):
        want, spread, size = attention(c.q[b].astype(np.float64), c.values["k"][b], c.values["v"][b], c.position[b], c.first[b],
                                       c.end[b], float(np.float32(scale)), c.cap, slopes)
        visible = np.broadcast_to((c.end - c.first)[b][:, None].astype(np.float64), size.shape)
        reach = 0.0 if slopes is None else np.abs(c.position[b])[:, None] * slopes[None, :]
        assert np.all(np.abs(got[b] - want) <= tolerance(want, spread, size, visible, 128, WEIGHTS["prompt"], 2.0 ** -24, c.cap, reach))


@pytest.mark.parametrize("cap", [30.0, 54.0])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("power", [60, -90])
@pytest.mark.parametrize("rows,path,fields", [(130, "prompt", {}), (130, "prompt", dict(ranges=True)), (2, "decode_bf16", {}),
                                              (2, "decode_codes", dict(cache=E4M3, page=64)), (9, "general", {})])
@pytest.mark.parametrize("chunk", [None, 128])
def test_large_and_small_values_under_logits_at_the_cap(backend, cap, sign, power, rows, path, fields, chunk):
    # every logit near the cap (or near its negative) and values of 10^18 or 10^-27: the answer is a mean of values
    fields = dict(fields)
    if fields.get("ranges"):
        fields["ranges"] = runs(2, [(0, 2 * i + 1) for i in range(rows)])
    c = Case(50, [400, 390], rows, 4, 2, 128, cap=cap, q_scale=40.0, **fields)
    c.q = np.abs(c.q)
    for x in (c.arrays, c.values):
        if c.cache:
            continue
        x["k"] = sign * np.abs(x["k"])
        x["v"] = x["v"] * np.float32(2.0 ** power)
    if c.cache:
        c.arrays["v_scales"] *= 2.0 ** power
        c.values["v"] *= 2.0 ** power
    c.check(backend, path, force_general=path == "general", chunk=chunk)


def test_logits_that_grow_along_the_sequence_under_a_cap(backend):
    # a prompt's tiles are walked from the last one: the reference of a row has to follow in both directions
    for direction in (1, -1):
        c = Case(51, [1500], 140, 2, 1, 128, cap=54.0, q_scale=1.0)
        ramp = (np.linspace(-45.0, 45.0, 1500)[::direction, None, None] / np.sqrt(128)).astype(np.float32)
        c.q[:] = 1.0
        for x in (c.arrays, c.values):
            x["k"] = np.where(np.isnan(x["k"]), np.nan, ramp[None] * np.ones_like(x["k"]))
        rounded = clori_b200.bf16_bits_to_f32(clori_b200.f32_to_bf16_bits(c.arrays["k"].astype(np.float32)))
        c.arrays["k"] = rounded
        c.values["k"] = np.nan_to_num(rounded).astype(np.float64)
        c.check(backend, "prompt")


FAR = [(1, "decode_bf16", {}), (3, "decode_codes", dict(cache=E4M3, page=64)), (70, "prompt", {}), (70, "prompt", dict(cap=20.0)),
       (50, "prompt", dict(cache=I8, page=16)), (5, "general", {}), (5, "general", dict(cap=9.0, kv_dtype=F32, q_dtype=F32))]


def check_far(backend, c, path, chunk):
    got, status = c.launch(backend, c.plan(backend, c.problem(backend, path == "general"), chunk))
    assert status == 0
    for b in range(len(c.lengths)):
        want, spread, size = attention(c.q[b].astype(np.float64), c.values["k"][b], c.values["v"][b], c.position[b], c.first[b],
                                       c.end[b], float(np.float32(1 / np.sqrt(128))), c.cap, c.slope.astype(np.float64))
        visible = (c.end - c.first)[b][:, None].astype(np.float64)
        # a softmax does not change when a row's logits all move: only distances among the tokens that it sees count
        allowed = tolerance(want, spread, size, np.broadcast_to(visible, size.shape), 128, WEIGHTS[path], 2.0 ** -24, c.cap,
                            visible * c.slope[None, :].astype(np.float64))
        assert np.all(np.abs(got[b] - want) <= allowed), float((np.abs(got[b] - want) / allowed).max())


@pytest.mark.parametrize("start", [[2 ** 31 - 200, 2 ** 30 + 77], [2 ** 24 + 5, 70000]])
@pytest.mark.parametrize("rows,path,fields", FAR)
@pytest.mark.parametrize("chunk", [None, 128])
def test_a_bias_far_behind_the_cache(backend, start, rows, path, fields, chunk):
    check_far(backend, Case(52, [300, 257], rows, 4, 2, 128, slopes=True, query_start=start, **fields), path, chunk)


@pytest.mark.parametrize("rows,path,fields", FAR)
@pytest.mark.parametrize("chunk", [None, 128])
def test_a_bias_in_front_of_what_a_row_sees(backend, rows, path, fields, chunk):
    c = Case(53, [700, 650], rows, 4, 2, 128, slopes=True, query_start=[0, 5], ranges=runs(2, [(300 + i, 640) for i in range(rows)]), **fields)
    check_far(backend, c, path, chunk)


@pytest.mark.parametrize("fields", [{}, dict(slopes=True), dict(cap=20.0), dict(cache=E4M3, page=64)])
@pytest.mark.parametrize("chunk", [None, 1280])
def test_padding_of_nan_inside_a_long_run(backend, fields, chunk):
    # few tokens that no row sees between the runs of many rows over a long cache: values and keys there are NaN
    rows, tokens = 40, 6000
    spans = [(17 * i, 2900 - i) if i % 2 else (2911 + i, tokens - i) for i in range(rows)]
    c = Case(54, [tokens], rows, 4, 2, 128, ranges=runs(1, spans), **fields)
    assert not c.seen[0].all() and c.seen[0, 2950]
    c.check(backend, "prompt", chunk=chunk)


def test_padding_of_infinities_between_documents(backend):
    rng = np.random.default_rng(55)
    for trial in range(6):
        first, end = np.zeros((2, 300), int), np.zeros((2, 300), int)
        for b in range(2):
            at = 0
            while at < 300:
                n = int(rng.integers(1, 90))
                first[b, at:at + n], end[b, at:at + n] = at, np.minimum(np.arange(at, at + n) + 1, 300)[:300 - at]
                at += n + int(rng.integers(0, 40))
        c = Case(56 + trial, [300, 280], 300, 4, 2, 128, ranges=(first, end))
        for x in ("k", "v"):
            bad = np.isnan(c.arrays[x])
            c.arrays[x][bad] = np.where(rng.random(int(bad.sum())) < 0.5, np.inf, -np.inf)
        for chunk in (None, 128):
            c.check(backend, "prompt", chunk=chunk)


@pytest.mark.parametrize("chunk", [None, 128])
@pytest.mark.parametrize("cache,page", [(E4M3, 16), (I8, 64), (PLAIN, 16)])
@pytest.mark.parametrize("start", [None, [4000, 2980], [0, 2999]])
def test_staged_rows_of_a_window_begin_where_it_does(backend, cache, page, start, chunk):
    # sessions much longer than the window; rows at their end, in their middle, at their beginning and behind the cache
    Case(61, [5000, 3000], 40, 4, 2, 128, cache=cache, page=page, window=300, query_start=start).check(backend, "prompt", chunk=chunk)


def test_staged_rows_of_a_window_and_first_tokens(backend):
    c = Case(62, [3000, 2700], 40, 4, 2, 128, cache=E4M3, page=64, window=500, slopes=True)
    given = np.tile(np.arange(40) * 20 + 2400, (2, 1))
    c.first = np.minimum(np.maximum(c.first, given), c.end)
    p = c.problem(backend)
    p.row_first = backend.tensor("first", given.astype(np.int32)).data_ptr
    got, status = c.launch(backend, c.plan(backend, p))
    want, spread, size = c.answer()
    assert status == 0 and np.all(np.abs(got - want) <= c.allowed(want, spread, size, "prompt"))


@pytest.mark.parametrize("fields", [dict(cache=E4M3, page=64), dict(page=16), dict(cache=I8, page=16, ranges=True, slopes=True, out_dtype=BF16),
                                    dict(cache=E4M3, page=64, query_start=[100, 50, 0, 200, 10], cap=20.0)])
def test_sessions_whose_staged_rows_do_not_fit_together(backend, fields):
    # capacity for 524288 tokens a session: two sessions at a time in a workspace of 4 GiB, three groups
    fields = dict(fields)
    if fields.get("ranges"):
        first = np.random.default_rng(63).integers(0, 100, (5, 70))
        fields["ranges"] = (first, first + 150)
    c = Case(64, [300, 129, 0, 257, 64], 70, 8, 8, 128, **fields)
    c.table = np.pad(c.table, ((0, 0), (0, 524288 // c.page - c.table.shape[1])), constant_values=-1)
    p = c.problem(backend)
    p.kv_tokens_max = 524288
    p = c.plan(backend, p)
    n = C.c_uint()
    for _ in range(2):
        assert backend.lib.yvx_cuda_scored_attention(C.byref(p), backend.stream, C.byref(n)) == 0
        assert backend.lib.yvx_cuda_stream_synchronize(backend.stream) == 0
        assert n.value == 3 * 2 + (p.max_splits > 1) and int(c.status.read()[0]) == 0
        got = c.result()
        want, spread, size = c.answer()
        assert np.all(np.abs(got - want) <= c.allowed(want, spread, size, "prompt"))


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("fields", [{}, dict(slopes=True), dict(causal=False)])
@pytest.mark.parametrize("chunk", [None, 128])
def test_products_beyond_the_range_of_the_mask_are_reported(backend, sign, fields, chunk):
    # Q . K of +-2^107 for every token: the prompt kernel says that it cannot weigh them, the others give the mean of V
    c = Case(65, [300], 70, 4, 2, 128, garbage=False, **fields)
    c.q[:] = 2.0 ** 50
    for x in (c.arrays, c.values):
        x["k"][:] = sign * 2.0 ** 50
    assert c.launch(backend, c.plan(backend, c.problem(backend), chunk))[1] == 1
    c = Case(66, [300], 2, 4, 2, 128, garbage=False, causal=False)
    c.q[:] = 2.0 ** 50
    for x in (c.arrays, c.values):
        x["k"][:] = sign * 2.0 ** 50
    for general in (False, True):
        got, status = c.launch(backend, c.plan(backend, c.problem(backend, general)))
        mean = np.repeat(c.values["v"][0].mean(0), 2, axis=0)
        spread = np.repeat(np.abs(c.values["v"][0]).mean(0), 2, axis=0)
        assert status == 0 and np.all(np.abs(got[0] - mean) <= spread * (2.0 ** -16 + 300 * 2.0 ** -22))


def test_a_loud_negative_token_has_no_weight(backend):
    c = Case(67, [300], 70, 4, 2, 128, garbage=False)
    c.q[:] = 2.0 ** 50
    for x in (c.arrays, c.values):
        x["k"][:] = 0.0
        x["k"][0, 3] = -(2.0 ** 50)
    c.check(backend, "prompt")
