"""Scored attention and the 8-bit cache in float64, and the drivers of their shim entries (test infrastructure)."""
import ctypes as C
import math

import numpy as np

import clori_b200
from clori_b200 import abi

LIMIT = {abi.KV_E4M3: 448.0, abi.KV_I8: 127.0}


def bf16(x):
    return clori_b200.bf16_bits_to_f32(clori_b200.f32_to_bf16_bits(np.asarray(x, np.float32)))


def _e4m3_values():
    out = np.empty(256, np.float64)
    for byte in range(256):
        e, f = (byte >> 3) & 15, byte & 7
        v = f * 2.0 ** -9 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        out[byte] = math.nan if byte & 0x7f == 0x7f else v
        out[byte] *= -1 if byte & 0x80 else 1
    return out


E4M3 = _e4m3_values()


def decode(codes, code):
    """uint8 codes -> the values they stand for."""
    return E4M3[codes] if code == abi.KV_E4M3 else codes.view(np.int8).astype(np.float64)


def encode(x, code):
    """float64 values inside the code's range -> uint8 codes, nearest, ties to the even code."""
    x = np.asarray(x, np.float64)
    if code == abi.KV_I8:
        return np.rint(x).astype(np.int8).view(np.uint8)
    _, e = np.frexp(np.abs(x))
    step = 2.0 ** (np.maximum(e - 1, -6) - 3)
    grid = np.abs(np.rint(x / step) * step)
    order = np.argsort(E4M3[:127], kind="stable")
    at = order[np.searchsorted(E4M3[:127][order], grid)]
    return (at | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def power_scale(amax, code):
    """The smallest power of two s >= 2^-126 with amax <= s * limit."""
    if amax == 0:
        return 2.0 ** -126
    m, e = math.frexp(float(amax) / LIMIT[code])
    return 2.0 ** max(-126, e - 1 if m == 0.5 else e)


def attention(q, k, v, position, first, end, scale, cap=0.0, slopes=None):
    """One session in float64. q [rows, heads, hd]; k, v [tokens, kv_heads, hd]. Returns the output, the weighted mean of
    |v| and, per row and head, a bound of sum |q||k| * scale over the visible tokens."""
    rows, heads, hd = q.shape
    group = heads // k.shape[1] if k.shape[1] else 1
    out = np.zeros((rows, heads, hd))
    spread, size = np.zeros((rows, heads, hd)), np.zeros((rows, heads))
    for r in range(rows):
        lo, hi = int(first[r]), int(end[r])
        if hi <= lo:
            continue
        tokens = np.arange(lo, hi)
        for h in range(heads):
            kk, vv = k[lo:hi, h // group], v[lo:hi, h // group]
            z = scale * (kk @ q[r, h])
            if cap:
                z = cap * np.tanh(z / cap)
            if slopes is not None:
                z = z - slopes[h] * np.abs(position[r] - tokens)
            w = np.exp(z - z.max())
            w /= w.sum()
            out[r, h], spread[r, h] = w @ vv, w @ np.abs(vv)
            size[r, h] = scale * (np.abs(kk) @ np.abs(q[r, h])).max()
    return out, spread, size


# What the weights of the softmax are rounded to: half a step of the type they are carried in.
WEIGHTS = {"general": 2.0 ** -22, "decode_bf16": 2.0 ** -16, "decode_codes": 2.0 ** -11, "prompt": 2.0 ** -8}


def tolerance(want, spread, size, visible, hd, weights, out_half_step, cap=0.0, reach=0.0):
    """|got - want| allowed. A dot product of hd products in F32 is off by at most hd * 2^-23 of sum |q||k| (each addition
    half a step or a truncation); the cap's tanh by 2^-20 of the cap; the bias by 2^-23 of slope * distance. An error d of
    a logit changes a weight by the factor e^d, in the numerator and in the sum: 2 d of the weighted mean of |v|. A weight
    is rounded to `weights`; F32 sums of `visible` terms are off by visible * 2^-24 of their absolute sum (twice: values
    and weights), and exp2 by 2^-21. The result is rounded once."""
    d = size * hd * 2.0 ** -23 + cap * 2.0 ** -20 + reach * 2.0 ** -23 + 2.0 ** -22
    relative = 2 * d + weights + 2 * visible * 2.0 ** -24 + 2.0 ** -20
    return relative[..., None] * spread + out_half_step * (np.abs(want) + relative[..., None] * spread) + 1e-30


class Case:
    """A call: host arrays, their float64 answer, and the device buffers of the shim problem."""

    def __init__(self, seed, lengths, rows, heads, kv_heads, hd, *, cache=abi.KV_PLAIN, kv_dtype=abi.DTYPE_BF16,
                 q_dtype=abi.DTYPE_BF16, out_dtype=abi.DTYPE_F32, page=0, causal=True, cap=0.0, slopes=False, window=0,
                 ranges=None, query_start=None, q_scale=1.0, k_scale=1.0, garbage=True, kv_max=None, head_major=False,
                 pad=0, outlier=None):
        rng = np.random.default_rng(seed)
        self.__dict__.update(locals())
        self.lengths = np.asarray(lengths, np.int64)
        S, T = len(lengths), int(kv_max if kv_max is not None else max(1, max(lengths)))
        self.kv_max = T
        q = (rng.standard_normal((S, rows, heads, hd)) * q_scale).astype(np.float32)
        self.q = bf16(q) if q_dtype == abi.DTYPE_BF16 else q
        self.slope = (2.0 ** (-8.0 * (1 + np.arange(heads)) / heads)).astype(np.float32) if slopes else None
        start = self.lengths - rows if query_start is None else np.asarray(query_start, np.int64)
        self.position = start[:, None] + np.arange(rows)[None, :]
        n = self.lengths[:, None]
        first = np.zeros_like(self.position) if ranges is None else ranges[0].astype(np.int64)
        end = (np.minimum(self.position + 1, n) if causal else n + 0 * self.position) if ranges is None else ranges[1].astype(np.int64)
        if window:
            first = np.maximum(first, self.position + 1 - window)
        self.end = np.clip(end, 0, n)
        self.first = np.minimum(np.maximum(first, 0), self.end)
        self._cache(rng, S, T)

    def _cache(self, rng, S, T):
        page, H, hd, code = self.page, self.kv_heads, self.hd, self.cache
        seen = np.zeros((S, T), bool)          # tokens that some row of the call sees
        for b in range(S):
            for r in range(self.rows):
                seen[b, self.first[b, r]:self.end[b, r]] = True
        self.seen = seen
        if page:
            per = [-(-int(x) // page) for x in self.lengths]
            width = max(1, -(-T // page))
            order = rng.permutation(sum(per) + 2)
            self.pages = len(order)
            self.table = np.full((S, width), -1, np.int32)
            at = 0
            for b, m in enumerate(per):
                self.table[b, :m] = order[at:at + m]
                at += m
            shape = (self.pages, H, page, hd) if (code or self.head_major) else (self.pages, page, H, hd)
        else:
            self.table = None
            shape = (S, H, T, hd) if self.head_major else (S, T, H, hd)
        self.arrays, self.values = {}, {}
        for x in ("k", "v"):
            a = rng.standard_normal(shape).astype(np.float32)
            if x == "k":
                a *= self.k_scale
            if self.outlier and x == "k":
                a[..., ::16] *= self.outlier
            scales = None
            if code:
                a *= np.exp(rng.standard_normal((self.pages, H, 1, 1))).astype(np.float32)
                scales = np.array([[power_scale(np.abs(a[i, h]).max(), code) for h in range(H)] for i in range(self.pages)], np.float32)
                a = encode((a / scales[:, :, None, None]).astype(np.float64), code)
            elif self.kv_dtype == abi.DTYPE_BF16:
                a = bf16(a)
            rows = []
            for b in range(S):
                r = np.zeros((T, H, hd))
                for t in range(int(self.lengths[b])):
                    where = self._slot(b, t)
                    value = decode(a[where], code) * scales[where[0]][:, None].astype(np.float64) if code else a[where]
                    r[t] = value
                rows.append(r)
            self.values[x] = np.stack(rows)
            if self.garbage:                   # NaN wherever no row looks
                bad = np.ones(shape[:2] + shape[2:3], bool)
                for b in range(S):
                    for t in np.nonzero(seen[b])[0]:
                        where = self._slot(b, int(t))
                        bad[(where[0], where[1], where[2])] = False
                a[bad] = (0x7f if code == abi.KV_E4M3 else 0x80 if code else np.nan)
            self.arrays[x], self.arrays[x + "_scales"] = a, scales

    def _slot(self, b, t):
        every = slice(None)
        if self.page:
            i, j = int(self.table[b, t // self.page]), t % self.page
            return (i, every, j) if (self.cache or self.head_major) else (i, j, every)
        return (b, every, t) if self.head_major else (b, t, every)

    def answer(self):
        scale = np.float32(1.0 / math.sqrt(self.hd))
        got = [attention(self.q[b].astype(np.float64), self.values["k"][b], self.values["v"][b], self.position[b], self.first[b],
                         self.end[b], float(scale), self.cap, None if self.slope is None else self.slope.astype(np.float64))
               for b in range(len(self.lengths))]
        return [np.stack(x) for x in zip(*got)]

    def allowed(self, want, spread, size, path):
        step = {abi.DTYPE_F32: 2.0 ** -24, abi.DTYPE_BF16: 2.0 ** -8}[self.out_dtype]
        visible = np.broadcast_to((self.end - self.first)[:, :, None].astype(np.float64), size.shape)
        reach = 0.0
        if self.slope is not None:
            far = np.maximum(np.abs(self.position - self.first), np.abs(self.position - self.end + 1))
            reach = far[:, :, None] * self.slope[None, None, :].astype(np.float64)
        return tolerance(want, spread, size, visible, self.hd, WEIGHTS[path], step, self.cap, reach)

    def problem(self, backend, force_general=False):
        """The shim problem with its device buffers (kept alive by the backend)."""
        p, H, hd, page = abi.ScoredProblem(), self.kv_heads, self.hd, self.page
        S = len(self.lengths)
        up = lambda name, a, dtype=None: backend.tensor(name, a, dtype)
        q_stride = self.heads * hd + self.pad
        q = np.full((S, self.rows, q_stride), np.nan, np.float32)
        q[:, :, :self.heads * hd] = self.q.reshape(S, self.rows, -1)
        q = up("q", clori_b200.f32_to_bf16_bits(q) if self.q_dtype == abi.DTYPE_BF16 else q)
        p.sessions, p.query_rows, p.query_heads, p.kv_heads, p.head_dim = S, self.rows, self.heads, H, hd
        p.causal, p.scale, p.cap, p.window = int(self.causal), 1.0 / math.sqrt(hd), self.cap, self.window
        p.query_dtype, p.kv_dtype, p.output_dtype, p.kv_code = self.q_dtype, self.kv_dtype, self.out_dtype, self.cache
        p.query, p.query_row_stride, p.query_session_stride = q.data_ptr, q_stride, self.rows * q_stride
        for x in ("k", "v"):
            a = self.arrays[x]
            if not self.cache and self.kv_dtype == abi.DTYPE_BF16:
                a = clori_b200.f32_to_bf16_bits(a)
            t = up(x, a.view(np.int8) if self.cache else a)
            setattr(p, {"k": "key", "v": "value"}[x], t.data_ptr)
            if self.cache:
                setattr(p, {"k": "key_scales", "v": "value_scales"}[x], up(x + "s", self.arrays[x + "_scales"]).data_ptr)
        inner = page if page else self.arrays["k"].shape[2 if self.head_major else 1]
        head_major = bool(self.cache) or self.head_major
        p.key_token_stride = p.value_token_stride = hd if head_major else H * hd
        p.key_head_stride = p.value_head_stride = inner * hd if head_major else hd
        p.key_outer_stride = p.value_outer_stride = inner * H * hd
        if page:
            p.block_table, p.block_tokens = up("table", self.table).data_ptr, page
            p.block_table_stride, p.pool_blocks = self.table.shape[1], self.pages
        p.kv_tokens, p.kv_tokens_max = up("lens", self.lengths.astype(np.int32)).data_ptr, self.kv_max
        if self.query_start is None:
            p.query_start_from_end = 1
        else:
            p.query_start = up("start", np.asarray(self.query_start, np.int32)).data_ptr
        if self.ranges is not None:
            p.row_first = up("first", self.ranges[0].astype(np.int32)).data_ptr
            p.row_end = up("end", self.ranges[1].astype(np.int32)).data_ptr
        if self.slope is not None:
            p.slopes = up("slopes", self.slope).data_ptr
        p.force_general = int(force_general)
        self.status = up("status", np.zeros(1, np.int32))
        self.out = up("out", np.full((S, self.rows, self.heads * hd), 0x7fc0, np.uint16) if self.out_dtype == abi.DTYPE_BF16
                      else np.full((S, self.rows, self.heads * hd), np.nan, np.float32))
        p.output, p.status = self.out.data_ptr, self.status.data_ptr
        return p

    def plan(self, backend, p, chunk=None):
        backend.lib.yvx_cuda_scored_plan(C.byref(p), backend.sm_count)
        if chunk:
            p.chunk_tokens, p.max_splits = chunk, -(-(-(-self.kv_max // 64) * 64) // chunk)
        self.work = backend.alloc("work", abi.DTYPE_I8, (max(256, backend.lib.yvx_cuda_scored_workspace_bytes(C.byref(p))),))
        p.workspace, p.workspace_bytes = self.work.data_ptr, self.work.nbytes
        return p

    def launch(self, backend, p):
        n = C.c_uint()
        rc = backend.lib.yvx_cuda_scored_attention(C.byref(p), backend.stream, C.byref(n))
        assert rc == 0, backend.lib.yvx_cuda_last_error_text()
        assert backend.lib.yvx_cuda_stream_synchronize(backend.stream) == 0, backend.lib.yvx_cuda_last_error_text()
        return self.result(), int(self.status.read()[0])

    def result(self):
        got = self.out.read()
        if self.out_dtype == abi.DTYPE_BF16:
            got = clori_b200.bf16_bits_to_f32(got)
        return got.reshape(len(self.lengths), self.rows, self.heads, self.hd)

    def check(self, backend, path, force_general=False, chunk=None):
        p = self.plan(backend, self.problem(backend, force_general), chunk)
        got, status = self.launch(backend, p)
        assert status == 0
        want, spread, size = self.answer()
        off = np.abs(got - want)
        allowed = self.allowed(want, spread, size, path)
        assert np.all(off <= allowed), (float(off.max()), float((off / allowed).max()))
        again, _ = self.launch(backend, p)
        assert np.array_equal(got, again)
        return p


def documents(lengths_per_session, rows, prefix=None):
    """row_first / row_end of sessions of packed documents."""
    out = [clori_b200.row_ranges(lengths, rows, 0, prefix) for lengths in lengths_per_session]
    return np.stack([x[0] for x in out]), np.stack([x[1] for x in out])
