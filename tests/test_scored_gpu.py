"""Scored attention on a B200 against float64: caps, distance bias, windows, visible runs, caches of every kind. What no
row sees holds NaN in every case; results repeat bit for bit; tolerances are derived in scored_cases.tolerance."""
import numpy as np
import pytest

import clori_b200
from clori_b200 import abi
from tests.scored_cases import WEIGHTS, Case, attention, documents, tolerance

pytestmark = pytest.mark.gpu
E4M3, I8, PLAIN = abi.KV_E4M3, abi.KV_I8, abi.KV_PLAIN
F32, BF16 = abi.DTYPE_F32, abi.DTYPE_BF16


GENERAL = [
    # lengths, rows, heads, kv_heads, hd, fields
    ([1], 1, 1, 1, 128, {}),
    ([0, 1, 33, 300], 1, 8, 2, 128, dict(kv_dtype=F32, q_dtype=F32)),
    ([5, 70, 129], 3, 6, 3, 64, dict(cap=20.0, q_scale=6.0)),
    ([200, 31], 5, 4, 1, 80, dict(slopes=True, out_dtype=BF16)),
    ([100, 257], 17, 4, 4, 256, dict(kv_dtype=F32, q_dtype=F32, slopes=True, cap=5.0, q_scale=3.0)),
    ([90, 90], 90, 5, 1, 40, dict(causal=False, slopes=True)),
    ([300, 129, 64], 4, 8, 2, 128, dict(page=16, window=70)),
    ([300, 129, 64], 2, 5, 1, 96, dict(page=48, kv_dtype=F32)),
    ([64, 130, 1], 2, 8, 2, 64, dict(cache=E4M3, page=16, cap=30.0, q_scale=4.0)),
    ([64, 130, 1], 2, 8, 2, 128, dict(cache=I8, page=24, slopes=True)),
    ([33], 33, 2, 2, 16, dict(cache=E4M3, page=7, pad=3)),
    ([40, 41], 8, 4, 2, 33, dict(head_major=True, window=5, pad=1)),
]


@pytest.mark.parametrize("lengths,rows,heads,kv_heads,hd,fields", GENERAL)
@pytest.mark.parametrize("chunk", [None, 64])
def test_general_kernel(backend, lengths, rows, heads, kv_heads, hd, fields, chunk):
    Case(11, lengths, rows, heads, kv_heads, hd, **fields).check(backend, "general", force_general=True, chunk=chunk)


LENGTHS = [1, 15, 16, 17, 63, 64, 65, 130, 0, 700]
DECODE = [
    # lengths, rows, heads, kv_heads, fields
    ([1], 1, 1, 1, {}),
    (LENGTHS, 1, 8, 2, dict(page=64)),
    (LENGTHS, 1, 5, 1, dict(page=128, cap=30.0, q_scale=6.0)),
    (LENGTHS, 3, 8, 2, dict(out_dtype=BF16, slopes=True)),
    ([500, 333], 4, 16, 2, dict(head_major=True, window=100)),
    ([500, 333], 2, 16, 1, dict(causal=False, slopes=True, cap=5.0, pad=8)),
    (LENGTHS, 1, 8, 2, dict(cache=E4M3, page=64)),
    (LENGTHS, 4, 4, 1, dict(cache=E4M3, page=16, cap=50.0, q_scale=8.0)),
    (LENGTHS, 1, 10, 2, dict(cache=I8, page=32, slopes=True, out_dtype=BF16)),
    (LENGTHS, 8, 16, 2, dict(cache=I8, page=128, window=90, cap=2.0)),
    (LENGTHS, 2, 2, 2, dict(cache=E4M3, page=64, q_scale=1e-30, k_scale=1e20)),
    ([200, 129], 3, 4, 2, dict(cache=E4M3, page=16, q_scale=3e5, k_scale=1e-7, outlier=40.0)),
    ([900, 64], 1, 4, 2, dict(cache=I8, page=64, query_start=[1000, 20])),
]


@pytest.mark.parametrize("lengths,rows,heads,kv_heads,fields", DECODE)
@pytest.mark.parametrize("chunk", [None, 64, 128])
def test_decode_kernel(backend, lengths, rows, heads, kv_heads, fields, chunk):
    path = "decode_codes" if fields.get("cache") else "decode_bf16"
    Case(12, lengths, rows, heads, kv_heads, 128, **fields).check(backend, path, chunk=chunk)


LOUDNESS = np.repeat(np.float32([0.02, 8.0, 1.0, 40.0, 0.1]), 128)[None, :, None, None]   # of keys, tile by tile
DOCS = [[100, 1, 130, 300, 0, 69]]
PROMPT = [
    # lengths, rows, heads, kv_heads, fields
    ([130], 130, 2, 1, {}),
    ([300, 257], 200, 2, 2, dict(out_dtype=BF16)),
    ([129, 70], 70, 4, 4, dict(cap=50.0, q_scale=3.0)),
    ([400, 390], 300, 2, 1, dict(cap=2.0, q_scale=8.0)),              # scores far outside the polynomial
    ([300], 300, 4, 2, dict(slopes=True)),
    ([520, 500], 500, 2, 1, dict(slopes=True, cap=20.0, q_scale=4.0, causal=False)),
    ([600], 600, 2, 1, dict(ranges="documents")),
    ([600], 600, 2, 1, dict(ranges="documents", slopes=True, cap=20.0)),
    ([600], 600, 2, 1, dict(ranges="prefix", slopes=True)),
    ([700, 650], 270, 2, 1, dict(window=140)),
    ([700, 300], 90, 4, 2, dict(window=300, page=64)),
    ([700, 300], 90, 4, 2, dict(page=128, pad=8, slopes=True)),
    ([300, 290], 280, 2, 1, dict(head_major=True, kv_max=513, cap=5.0)),
    ([300, 200], 150, 2, 1, dict(query_start=[10, 300])),
    ([390, 261], 200, 4, 2, dict(cache=E4M3, page=64)),
    ([390, 261], 200, 4, 2, dict(cache=I8, page=16, window=90, cap=9.0, q_scale=4.0)),
    ([200, 210], 130, 2, 1, dict(page=16)),
    ([0, 300], 257, 2, 1, {}),
    # groups that fill a row tile, that leave rows of it unused, and one that no tile holds
    ([500, 333], 8, 16, 2, dict(head_major=True, window=100)),
    ([700, 0, 129], 11, 6, 2, dict(page=64, slopes=True)),
    ([260, 300], 60, 10, 2, dict(cap=30.0, q_scale=3.0, out_dtype=BF16)),
    ([300, 260], 33, 14, 2, dict(ranges="prefix", slopes=True, cap=4.0)),
    ([200, 130], 10, 65, 1, dict(causal=False)),
    ([200, 130], 2, 129, 1, dict(slopes=True)),
    ([1000, 900], 9, 16, 2, dict(cache=E4M3, page=64, cap=30.0, q_scale=6.0)),
    # caps: every form of tanh in turn, logits far below zero everywhere, caps beyond the fixed reference
    ([640], 200, 2, 1, dict(cap=20.0, k_scale=LOUDNESS)),
    ([400, 390], 130, 2, 1, dict(cap=54.0, q_scale=60.0)),
    ([400, 390], 130, 2, 1, dict(cap=300.0, q_scale=60.0)),
    ([400, 390], 130, 2, 1, dict(cap=300.0, q_scale=60.0, slopes=True)),
]


@pytest.mark.parametrize("lengths,rows,heads,kv_heads,fields", PROMPT)
@pytest.mark.parametrize("chunk", [None, 128, 384])
def test_prompt_kernel(backend, lengths, rows, heads, kv_heads, fields, chunk):
    fields = dict(fields)
    if fields.get("ranges") == "documents":
        fields["ranges"] = documents(DOCS, rows)
    elif fields.get("ranges") == "prefix":
        fields["ranges"] = documents([[rows]] * len(lengths), rows, [min(250, rows // 2)])
    Case(14, lengths, rows, heads, kv_heads, 128, **fields).check(backend, "prompt", chunk=chunk)


def test_prompt_rows_with_gaps_and_padding(backend):
    # packed documents with padding between them: keys and values of the padding are NaN
    first, end = np.zeros((1, 400), int), np.zeros((1, 400), int)
    for lo, hi in ((0, 90), (100, 101), (140, 330), (350, 390)):
        first[0, lo:hi], end[0, lo:hi] = lo, np.arange(lo, hi) + 1
    for chunk in (None, 128, 256):
        Case(15, [400], 400, 2, 1, 128, ranges=(first, end)).check(backend, "prompt", chunk=chunk)
        Case(15, [400], 400, 2, 1, 128, ranges=(first, end), cache=E4M3, page=64, slopes=True).check(backend, "prompt", chunk=chunk)


def test_pages_in_front_of_a_window_may_be_gone(backend):
    for rows, fields in ((1, dict(cache=E4M3, page=16)), (1, dict(page=64)), (100, dict(cache=I8, page=16)), (100, dict(page=64)),
                         (100, dict(page=16))):
        for general in (False, True):
            c = Case(16, [700, 650], rows, 4, 2, 128, window=50, **fields)
            for b in range(2):
                c.table[b, :int(c.first[b].min()) // c.page] = -1
            got, status = c.launch(backend, c.plan(backend, c.problem(backend, general)))
            want, spread, size = c.answer()
            assert status == 0 and np.all(np.abs(got - want) <= c.allowed(want, spread, size, "prompt"))


def test_one_loud_token_does_not_hide_many_quiet_ones(backend):
    # weights far below the largest carry half of the result: they have to survive their rounding
    for fields, path in ((dict(page=64), "decode_bf16"), (dict(cache=E4M3, page=64), "decode_codes")):
        c = Case(13, [6000], 1, 2, 1, 128, q_scale=0.0, garbage=False, **fields)
        c.slope = np.array([0.0, 0.0], np.float32)
        c.q[:] = 1.0
        a, s = c.arrays["k"], c.arrays["k_scales"]
        block, slot = int(c.table[0, 0]), 3
        if fields.get("cache"):
            a[:], s[:] = 0, 2.0 ** -126
            s[block] = 1.0
            a[block, :, slot] = 0x38            # 1.0 in every lane: the score is sqrt(128), 2^16 times the others' weight
            c.values["k"][:] = 0.0
        else:
            a[:] = 0.0
            a[block, slot] = 1.0
            c.values["k"][:] = 0.0
        c.values["k"][0, 3] = 1.0
        c.check(backend, path)


@pytest.mark.parametrize("sessions,rows,heads,kv_heads,hd,fields", [
    (256, 1, 8, 2, 128, dict(page=16)), (300, 1, 7, 7, 33, dict(kv_dtype=F32)), (40, 13, 4, 2, 128, dict(out_dtype=BF16)),
])
def test_many_items_of_few_splits(backend, sessions, rows, heads, kv_heads, hd, fields):
    lengths = [(37 * i) % 200 for i in range(sessions)]
    for chunk, general in ((64, False), (64, True)):
        path = "general" if general or hd != 128 else "decode_bf16"
        Case(31, lengths, rows, heads, kv_heads, hd, **fields).check(backend, path, force_general=general, chunk=chunk)


@pytest.mark.parametrize("cap,loud", [(300.0, 50.0), (300.0, 44.0), (1000.0, 150.0), (50.0, 7.0), (5.0, 0.6), (0.01, 0.0013)])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("rows,path", [(70, "prompt"), (2, "decode_bf16"), (5, "general")])
def test_the_whole_curve_of_a_cap(backend, cap, loud, slopes, rows, path):
    # products of one sign: logits around the cap and no cancellation that would hide an error of the tanh
    c = Case(34, [300, 280], rows, 4, 2, 128, cap=cap, q_scale=loud, slopes=slopes)
    c.q = np.abs(c.q)
    for x in (c.arrays, c.values):
        x["k"] = np.abs(x["k"])
    c.check(backend, path, force_general=path == "general")


@pytest.mark.parametrize("fields", [{}, dict(cap=20.0, q_scale=4.0), dict(slopes=True, page=64), dict(ranges=True), dict(ranges=True, cap=9.0, slopes=True)])
@pytest.mark.parametrize("chunk", [None, 128])
def test_many_pieces_of_work(backend, fields, chunk):
    # several pieces for every SM, empty ones and sessions of length 0 among them, against the F32 kernel; its result over
    # |v| is the weighted mean of |v| that a weight's rounding (half a step of bf16) is a part of
    fields, rng = dict(fields), np.random.default_rng(35)
    rows, sessions = 100, 70
    lengths = rng.integers(0, 420, sessions) * (rng.random(sessions) > 0.2)
    if fields.pop("ranges", False):
        end = rng.integers(0, 420, (sessions, rows))
        fields["ranges"] = (np.maximum(0, end - rng.integers(1, 300, (sessions, rows))) * (rng.random((sessions, rows)) > 0.3), end)
        fields["ranges"][1][rng.random(sessions) < 0.2] = 0

    c = Case(36, lengths, rows, 8, 2, 128, garbage=False, kv_max=420, **fields)

    def run(general):
        got, status = c.launch(backend, c.plan(backend, c.problem(backend, general), chunk))
        assert status == 0
        return got

    got, again, want = run(False), run(False), run(True)
    c.arrays["v"] = np.abs(c.arrays["v"])
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * 1.05 * run(True) + 1e-6)
    assert np.array_equal(got, again)


@pytest.mark.parametrize("scale,cap", [(1e-14, 0.0), (1e-10, 0.0), (3e-5, 1e-4), (20.0, 60.0)])
def test_extreme_scales_with_a_bias(backend, scale, cap):
    c = Case(33, [300, 290], 70, 4, 2, 128, slopes=True, cap=cap, k_scale=min(1.0, 1e-2 / scale) if scale > 1 else 1.0)
    p = c.problem(backend)
    p.scale = scale
    got, status = c.launch(backend, c.plan(backend, p))
    assert status == 0
    for b in range(2):
        want, spread, size = attention(c.q[b].astype(np.float64), c.values["k"][b], c.values["v"][b], c.position[b], c.first[b],
                                       c.end[b], float(np.float32(scale)), float(np.float32(cap)), c.slope.astype(np.float64))
        visible = np.broadcast_to((c.end - c.first)[b][:, None].astype(np.float64), size.shape)
        reach = np.abs(c.position[b])[:, None] * c.slope[None, :].astype(np.float64)
        assert np.all(np.abs(got[b] - want) <= tolerance(want, spread, size, visible, 128, WEIGHTS["prompt"], 2.0 ** -24, cap, reach))


def test_rows_in_front_of_the_session_and_empty_sessions_are_zero(backend):
    c = Case(5, [2, 0, 7], 4, 4, 2, 128)
    p = c.plan(backend, c.problem(backend))
    got, status = c.launch(backend, p)
    assert status == 0
    assert not got[0, :2].any() and got[0, 2:].any() and not got[1].any() and got[2].any()


def test_row_runs_with_gaps_padding_and_reversed_bounds(backend):
    rng = np.random.default_rng(3)
    first = rng.integers(-5, 180, (2, 9))
    end = first + rng.integers(-20, 80, (2, 9))
    c = Case(6, [190, 150], 9, 4, 2, 128, ranges=(first, end), slopes=True)
    for general in (False, True):
        c.check(backend, "general" if general else "decode_bf16", force_general=general)


def test_a_nan_that_is_seen_is_reported(backend):
    for x in ("k", "v"):
        for fields in (dict(), dict(kv_dtype=F32, q_dtype=F32)):
            c = Case(7, [100], 1, 4, 2, 128, garbage=False, **fields)
            c.arrays[x][0, 50] = np.nan
            assert c.launch(backend, c.plan(backend, c.problem(backend)))[1] == 1


@pytest.mark.parametrize("fields", [dict(), dict(cap=10.0), dict(slopes=True), dict(cap=10.0, slopes=True)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_nan_that_a_prompt_row_sees_is_reported(backend, fields, value):
    # in a tile that every row sees whole, in one that the causal mask cuts, and for the last row alone
    for token in (50, 250, 299):
        for x in ("k", "v"):
            c = Case(7, [300], 300, 2, 1, 128, garbage=False, **fields)
            c.arrays[x][0, token] = value
            if x == "k" and value == np.inf and fields.get("cap"):
                continue                        # a cap makes an infinite product finite
            assert c.launch(backend, c.plan(backend, c.problem(backend)))[1] == 1, (token, x)


def test_bad_lengths_and_table_entries_are_reported(backend):
    c = Case(8, [100, 90], 1, 4, 2, 128, page=64, cache=E4M3)
    c.table[1, 0] = 9999
    assert c.launch(backend, c.plan(backend, c.problem(backend)))[1] == 2
    c = Case(8, [100, 90], 1, 4, 2, 128, page=64)
    p = c.plan(backend, c.problem(backend))
    too_long = backend.tensor("lens", np.array([100, 2000], np.int32))
    p.kv_tokens = too_long.data_ptr
    got, status = c.launch(backend, p)
    assert status == 2 and not got[1].any()
