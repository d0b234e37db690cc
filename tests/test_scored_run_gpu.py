"""The 8-bit cache, its page bookkeeping, page copies and scored attention together as a serving loop uses them, the
operator level of scored attention, and captured, repeated and asynchronous calls."""
import ctypes as C

import numpy as np
import pytest

import clori_b200
from clori_b200 import abi
from tests.scored_cases import WEIGHTS, Case, attention, bf16, decode, tolerance

pytestmark = pytest.mark.gpu
E4M3, I8, PLAIN = abi.KV_E4M3, abi.KV_I8, abi.KV_PLAIN
F32, BF16 = abi.DTYPE_F32, abi.DTYPE_BF16
HEADS, KV_HEADS, HD, PAGE, PAGES, PER = 8, 2, 128, 16, 40, 16


class Serving:
    """One layer's cache of codes and the calls of a serving loop on it."""

    def __init__(self, backend, code, cap, slopes):
        self.backend, self.code, self.cap = backend, code, cap
        self.rng = np.random.default_rng(90)
        self.slopes = np.exp2(-np.arange(1.0, HEADS + 1)).astype(np.float32) if slopes else None
        self.pool = clori_b200.KvPool(PAGES, PAGE, 8, PER)
        shape = (PAGES, KV_HEADS, PAGE, HD)
        # pages that were never written hold whatever the memory held: NaN codes and scales here
        self.codes = [backend.tensor(x, np.full(shape, 0x7f, np.int8)) for x in "kv"]
        self.scales = [backend.tensor(x, np.full(shape[:2], np.nan, np.float32)) for x in "st"]

    def rows(self, *shape):
        return bf16(self.rng.standard_normal(shape) * np.exp(self.rng.standard_normal(shape[:1] + (1,) * (len(shape) - 1))))

    def tables(self, sessions):
        return self.backend.tensor("table", np.stack([self.pool.table(s) for s in sessions]))

    def lengths(self, values):
        return self.backend.tensor("n", np.array(values, np.int32))

    def copy(self, copies):
        if copies:
            self.backend.kv_pages_copy([(t, KV_HEADS) for t in self.codes] + [(t, None) for t in self.scales], copies, PAGE)

    def append(self, sessions, fresh):
        """Reserve, make shared pages private, write and commit `fresh[i]` rows of session i."""
        n = max(fresh)
        present = [self.pool.committed(s) for s in sessions]
        self.copy([c for s, f in zip(sessions, fresh) for c in [self.pool.reserve(s, f)] if c])
        new = [clori_b200.f32_to_bf16_bits(self.rows(len(sessions), n, KV_HEADS * HD)) for _ in range(2)]
        up = self.backend.tensor
        self.backend.kv8_append(up("nk", new[0]), up("nv", new[1]), *self.codes, *self.scales, self.tables(sessions),
                                kv_code=self.code, max_kv_tokens=max(present), kv_tokens=self.lengths(present),
                                new_tokens=self.lengths(fresh))
        for s, f in zip(sessions, fresh):
            self.pool.commit(s, f)

    def attend(self, sessions, rows, check=True):
        """The last `rows` tokens of each session against its cache; compared with float64 over the codes."""
        n = [self.pool.committed(s) for s in sessions]
        q = self.rows(len(sessions), rows, HEADS * HD)
        up = self.backend.tensor
        out = up("o", np.zeros((len(sessions), rows, HEADS * HD), np.float32))
        slopes = None if self.slopes is None else up("w", self.slopes)
        again = lambda: self.backend.attention_scored(
            up("q", clori_b200.f32_to_bf16_bits(q)), *self.codes, self.lengths(n), out, kv_heads=KV_HEADS, head_dim=HD,
            max_kv_tokens=PER * PAGE, score_cap=self.cap, slopes=slopes, kv_code=self.code, key_scales=self.scales[0],
            value_scales=self.scales[1], block_table=self.tables(sessions), block_tokens=PAGE)
        assert again()[1].kernel_launches >= 1
        got = out.read().reshape(len(sessions), rows, HEADS, HD)
        codes, scales = [t.read() for t in self.codes], [t.read() for t in self.scales]
        path = "prompt" if rows * (HEADS // KV_HEADS) > 64 else "decode_codes"
        for i, s in enumerate(sessions):
            table = self.pool.table(s)[:-(-n[i] // PAGE)]
            k, v = [np.concatenate([(decode(c[p].view(np.uint8), self.code) * a[p][:, None, None]).transpose(1, 0, 2) for p in table])[:n[i]]
                    for c, a in zip(codes, scales)]
            position = n[i] - rows + np.arange(rows)
            end = np.clip(position + 1, 0, n[i])
            slope = None if self.slopes is None else self.slopes.astype(np.float64)
            want, spread, size = attention(q[i].reshape(rows, HEADS, HD).astype(np.float64), k, v, position, 0 * end, end,
                                           float(np.float32(1 / np.sqrt(HD))), self.cap, slope)
            reach = 0.0 if slope is None else n[i] * slope[None, :]
            allowed = tolerance(want, spread, size, end[:, None].astype(np.float64), HD, WEIGHTS[path], 2.0 ** -24, self.cap, reach)
            assert np.all(np.abs(got[i] - want) <= allowed), (s, float((np.abs(got[i] - want) / allowed).max()))
        return got, again, out


@pytest.mark.parametrize("code,cap,slopes", [(E4M3, 0.0, False), (I8, 30.0, False), (E4M3, 5.0, True)])
def test_a_serving_loop(backend, code, cap, slopes):
    s = Serving(backend, code, cap, slopes)
    a, b = s.pool.open(), s.pool.open()
    s.append([a, b], [75, 40])                       # prompts that end inside pages
    s.attend([a], 75)
    s.attend([b], 40)
    for _ in range(3):                               # a step of the batch
        s.append([a, b], [1, 1])
        s.attend([a, b], 1)
    child = s.pool.fork(a)                           # both write on from a shared, partly filled page
    s.append([a, child, b], [5, 3, 1])
    s.attend([a, child, b], 3)
    s.append([child], [6])                           # six drafted tokens, two of them accepted
    s.attend([child], 6)
    s.pool.truncate(child, s.pool.committed(child) - 4)
    s.append([a, child], [1, 17])
    got, again, out = s.attend([child, a, b], 2)
    s.pool.close_session(b)                          # its pages leave holes, the others move to the front
    got, again, out = s.attend([child, a], 2)
    before = s.pool.free_blocks()
    copies = s.pool.compact()
    assert copies and s.pool.free_blocks() == before
    s.copy(copies)
    used = PAGES - before
    assert all(s.pool.table(x)[:-(-s.pool.committed(x) // PAGE)].max() < used for x in (a, child))
    again()
    assert np.array_equal(out.read().reshape(got.shape), got)       # the same codes: the same bits
    s.append([a, child], [20, 1])
    s.attend([child, a], 4)
    s.attend([a], 33)
    s.pool.destroy()


def call(backend, sessions, rows, tokens, *, dtype=np.uint16, hd=HD, out=np.float32, seed=3, **fields):
    rng = np.random.default_rng(seed)
    bits = lambda x: clori_b200.f32_to_bf16_bits(x) if dtype is np.uint16 else x
    values = [bf16(rng.standard_normal(s)) for s in ((sessions, rows, HEADS * hd), (sessions, tokens, KV_HEADS * hd),
                                                     (sessions, tokens, KV_HEADS * hd))]
    q, k, v = [backend.tensor(n, bits(x)) for n, x in zip("qkv", values)]
    o = backend.tensor("o", np.zeros((sessions, rows, HEADS * hd), out))
    n = rng.integers(rows, tokens + 1, sessions).astype(np.int32)
    return values, n, (q, k, v, backend.tensor("n", n), o), dict(dict(
        kv_heads=KV_HEADS, head_dim=hd, max_kv_tokens=tokens, kv_outer_stride=tokens * KV_HEADS * hd), **fields)


@pytest.mark.parametrize("rows,tokens,hd,dtype,path", [(1, 90, 128, np.uint16, "decode_bf16"), (40, 200, 128, np.uint16, "prompt"),
                                                       (3, 70, 64, np.float32, "general")])
def test_operator_over_contiguous_rows(backend, rows, tokens, hd, dtype, path):
    (q, k, v), n, args, fields = call(backend, 3, rows, tokens, hd=hd, dtype=dtype)
    rc, facts = backend.attention_scored(*args, score_cap=7.0, window=50, **fields)
    assert rc == 0 and facts.kernel_launches >= 1
    got = args[4].read().reshape(3, rows, HEADS, hd)
    for b in range(3):
        position = n[b] - rows + np.arange(rows)
        end = position + 1
        first = np.maximum(0, end - 50)
        want, spread, size = attention(q[b].reshape(rows, HEADS, hd).astype(np.float64), k[b].reshape(tokens, KV_HEADS, hd).astype(np.float64),
                                       v[b].reshape(tokens, KV_HEADS, hd).astype(np.float64), position, first, end,
                                       float(np.float32(1 / np.sqrt(hd))), 7.0)
        allowed = tolerance(want, spread, size, (end - first)[:, None].astype(np.float64), hd, WEIGHTS[path], 2.0 ** -24, 7.0)
        assert np.all(np.abs(got[b] - want) <= allowed)


def test_operator_refusals(backend):
    _, _, args, fields = call(backend, 2, 4, 64)
    q, k, v, n, o = args
    run = lambda *a, **f: backend.attention_scored(*(a or args), check=False, **dict(fields, **f))[0]
    assert run() == 0
    assert run(kv_heads=3) == abi.YVEX_ERR_INVALID_ARG
    assert run(score_cap=-1.0) == abi.YVEX_ERR_INVALID_ARG
    assert run(score_cap=float("nan")) == abi.YVEX_ERR_INVALID_ARG
    assert run(scale=float("inf")) == abi.YVEX_ERR_INVALID_ARG
    assert run(kv_outer_stride=0) == abi.YVEX_ERR_INVALID_ARG
    assert run(query_token_stride=HEADS * HD - 1) == abi.YVEX_ERR_INVALID_ARG
    assert run(kv_outer_stride=64 * KV_HEADS * HD + 1) == abi.YVEX_ERR_FORMAT
    assert run(max_kv_tokens=65) == abi.YVEX_ERR_FORMAT
    assert run(kv_token_stride=2 ** 62) == abi.YVEX_ERR_INVALID_ARG
    assert run(kv_code=E4M3) == abi.YVEX_ERR_UNSUPPORTED
    assert run(kv_code=9) == abi.YVEX_ERR_UNSUPPORTED
    assert run(max_kv_tokens=2 ** 31) == abi.YVEX_ERR_BOUNDS
    assert run(window=2 ** 33) == abi.YVEX_ERR_BOUNDS
    assert run(slopes=backend.tensor("s", np.zeros(HEADS - 1, np.float32))) == abi.YVEX_ERR_FORMAT
    assert run(row_end=backend.tensor("e", np.zeros(7, np.int32))) == abi.YVEX_ERR_FORMAT
    assert run(q, k, backend.tensor("f", np.zeros((2, 64, KV_HEADS * HD), np.float32)), n, o) == abi.YVEX_ERR_UNSUPPORTED
    assert run(q, k, v, n, backend.alloc("short", F32, (2, 3, HEADS * HD), 2 * 3 * HEADS * HD * 4)) == abi.YVEX_ERR_FORMAT
    assert run(backend.alloc("unwritten", BF16, (2, 4, HEADS * HD), 2 * 4 * HEADS * HD * 2), k, v, n, o) == abi.YVEX_ERR_FORMAT
    table = backend.tensor("t", np.zeros((2, 3), np.int32))
    assert run(block_table=table, block_tokens=16, kv_outer_stride=0) == abi.YVEX_ERR_INVALID_ARG    # covers 48 of 64 tokens
    with clori_b200.Backend(0) as other:
        assert run(q, k, v, other.tensor("n", np.array([64, 64], np.int32)), o) == abi.YVEX_ERR_FORMAT
    assert run() == 0


def capture(backend, *launches):
    """The launches as one graph; they see the buffers' contents at replay."""
    graph = C.c_void_p()
    assert backend.lib.yvx_cuda_graph_capture_begin(backend.stream) == 0
    for launch in launches:
        assert launch() == 0, backend.lib.yvx_cuda_last_error_text()
    assert backend.lib.yvx_cuda_graph_capture_end(backend.stream, C.byref(graph)) == 0
    return graph


def replay(backend, graph):
    assert backend.lib.yvx_cuda_graph_launch(graph, backend.stream) == 0
    assert backend.lib.yvx_cuda_stream_synchronize(backend.stream) == 0


CAPTURED = [
    ([700, 90], 1, 8, 2, 64, dict(page=64)),                         # split decode and its fold
    ([700, 90], 1, 8, 2, 64, dict(cache=E4M3, page=16, cap=20.0)),
    ([300, 290], 60, 8, 2, 128, dict(slopes=True)),                  # split prompt
    ([300, 290], 60, 8, 2, None, dict(cache=I8, page=16, cap=9.0)),  # staged prompt
    ([90, 31], 3, 6, 3, None, dict(kv_dtype=F32)),                   # general kernel
]


@pytest.mark.parametrize("lengths,rows,heads,kv_heads,chunk,fields", CAPTURED)
def test_captured_calls_follow_their_buffers(backend, lengths, rows, heads, kv_heads, chunk, fields):
    c = Case(21, lengths, rows, heads, kv_heads, 128, garbage=False, **fields)
    p = c.plan(backend, c.problem(backend), chunk)
    graph = capture(backend, lambda: backend.lib.yvx_cuda_scored_attention(C.byref(p), backend.stream, None))
    buffers = {t.data_ptr: t for t in backend._tensors}
    q, n = buffers[p.query], buffers[p.kv_tokens]
    first = q.read()
    for turn in range(3):
        q.write(first if turn != 1 else first[..., ::-1])
        n.write(np.array(lengths, np.int32) - 7 * turn)
        replay(backend, graph)
        got = c.result().copy()
        eager, status = c.launch(backend, p)
        assert status == 0 and np.array_equal(got, eager)
    backend.lib.yvx_cuda_graph_destroy(graph)


def test_two_captured_graphs_with_a_workspace_each_run_on_two_streams(backend):
    cases = [Case(22, [900, 500], 1, 8, 2, 128, page=64), Case(23, [400, 390], 60, 8, 2, 128, cache=E4M3, page=64)]
    problems = [c.plan(backend, c.problem(backend), 128) for c in cases]
    want = [c.launch(backend, p)[0].copy() for c, p in zip(cases, problems)]
    lib = backend.lib
    graphs = [capture(backend, lambda p=p: lib.yvx_cuda_scored_attention(C.byref(p), backend.stream, None)) for p in problems]
    streams = [C.c_void_p() for _ in cases]
    for s in streams:
        assert lib.yvx_cuda_stream_create(C.byref(s)) == 0
    for c in cases:
        c.out.write(np.full(c.out.shape, np.nan, np.float32))
    for _ in range(8):
        for g, s in zip(graphs, streams):
            assert lib.yvx_cuda_graph_launch(g, s) == 0
    for s in streams:
        assert lib.yvx_cuda_stream_synchronize(s) == 0
    for c, w in zip(cases, want):
        assert np.array_equal(c.result(), w)
    for g, s in zip(graphs, streams):
        lib.yvx_cuda_graph_destroy(g)
        assert lib.yvx_cuda_stream_destroy(s) == 0


def test_an_asynchronous_backend_reports_at_the_next_synchronisation(backend):
    stream = C.c_void_p()
    assert backend.lib.yvx_cuda_stream_create(C.byref(stream)) == 0
    _, _, args, fields = call(backend, 3, 20, 100, out=np.float32)
    backend.attention_scored(*args, **fields)
    want = args[4].read()
    backend.bind_stream(stream.value, synchronous=False)
    args[4].write(np.zeros_like(want))
    for _ in range(3):                              # several calls are joined without a wait between them
        backend.attention_scored(*args, **fields)
    backend.sync()
    assert np.array_equal(args[4].read(), want)
    args[3].write(np.array([50, 101, 50], np.int32))    # longer than the call allows
    backend.attention_scored(*args, **fields)
    with pytest.raises(clori_b200.YvexError):
        backend.sync()
    args[3].write(np.array([50, 60, 50], np.int32))
    backend.attention_scored(*args, **fields)
    backend.sync()
    backend.bind_stream(None)
    assert backend.lib.yvx_cuda_stream_destroy(stream) == 0


@pytest.mark.parametrize("code", [E4M3, I8])
def test_pages_that_lie_beyond_32_bits(backend, code):
    # five pages 2^30 bytes apart give, bit for bit, what they give side by side
    rng = np.random.default_rng(44)
    lib, n, table = backend.lib, 250, np.array([[4, 0, 3, 1]], np.int32)
    new = [backend.tensor(x, clori_b200.f32_to_bf16_bits(bf16(rng.standard_normal((n, KV_HEADS * HD))))) for x in "ab"]
    status = backend.tensor("status", np.zeros(1, np.int32))
    tables = [backend.tensor("t", t) for t in (table, np.array([[2, 0, 3, 1]], np.int32))]
    outputs = []
    for stride in (2 * KV_HEADS * 64 * HD, 2 ** 30):
        pool = backend.alloc("pool", abi.DTYPE_I8, (4 * stride + 2 * KV_HEADS * 64 * HD,))
        scales = [backend.tensor(x, np.zeros((5, KV_HEADS), np.float32)) for x in "ks"]
        a = abi.Kv8AppendArgs()
        a.sessions, a.tokens, a.kv_heads, a.head_dim, a.code, a.dtype = 1, n, KV_HEADS, HD, code, BF16
        a.key, a.value, a.token_stride, a.session_stride = new[0].data_ptr, new[1].data_ptr, KV_HEADS * HD, n * KV_HEADS * HD
        a.block_table, a.block_tokens, a.block_table_stride, a.pool_blocks = tables[0].data_ptr, 64, 4, 5
        a.key_codes, a.value_codes = pool.data_ptr, pool.data_ptr + KV_HEADS * 64 * HD
        a.code_token_stride, a.code_head_stride, a.code_block_stride = HD, 64 * HD, stride
        a.key_scales, a.value_scales, a.status = scales[0].data_ptr, scales[1].data_ptr, status.data_ptr
        assert lib.yvx_cuda_kv8_append(C.byref(a), backend.stream) == 0, lib.yvx_cuda_last_error_text()

        def attend(rows, general, pages):
            q = backend.tensor("q", clori_b200.f32_to_bf16_bits(bf16(np.random.default_rng(rows).standard_normal((rows, HEADS * HD)))))
            out = backend.tensor("o", np.full((rows, HEADS * HD), np.nan, np.float32))
            p = abi.ScoredProblem()
            p.sessions, p.query_rows, p.query_heads, p.kv_heads, p.head_dim, p.causal = 1, rows, HEADS, KV_HEADS, HD, 1
            p.scale, p.query_dtype, p.kv_dtype, p.output_dtype, p.kv_code = 0.1, BF16, abi.DTYPE_I8, F32, code
            p.query, p.query_row_stride, p.query_session_stride = q.data_ptr, HEADS * HD, rows * HEADS * HD
            p.output, p.key, p.value, p.status = out.data_ptr, a.key_codes, a.value_codes, status.data_ptr
            p.key_token_stride = p.value_token_stride = HD
            p.key_head_stride = p.value_head_stride = 64 * HD
            p.key_outer_stride = p.value_outer_stride = stride
            p.key_scales, p.value_scales = a.key_scales, a.value_scales
            p.block_table, p.block_tokens, p.block_table_stride, p.pool_blocks = pages.data_ptr, 64, 4, 5
            p.kv_tokens_uniform, p.kv_tokens_max, p.query_start_from_end, p.force_general = n, n, 1, general
            lib.yvx_cuda_scored_plan(C.byref(p), backend.sm_count)
            work = backend.alloc("work", abi.DTYPE_I8, (max(256, lib.yvx_cuda_scored_workspace_bytes(C.byref(p))),))
            p.workspace, p.workspace_bytes = work.data_ptr, work.nbytes
            assert lib.yvx_cuda_scored_attention(C.byref(p), backend.stream, None) == 0, lib.yvx_cuda_last_error_text()
            assert lib.yvx_cuda_stream_synchronize(backend.stream) == 0 and int(status.read()[0]) == 0
            return out.read()

        calls = [(1, 0), (1, 1), (40, 0), (40, 1)]
        got = [attend(*x, tables[0]) for x in calls]
        pools = (abi.KvPagePool * 3)(abi.KvPagePool(pool.data_ptr, stride, 64 * HD, HD, 0, 5, 2 * KV_HEADS),
                                     *[abi.KvPagePool(s.data_ptr, KV_HEADS * 4, 0, 0, KV_HEADS * 4, 5, 1) for s in scales])
        copies = (abi.KvCopy * 1)(abi.KvCopy(1, 4, 2, 64))
        c = abi.KvPagesArgs()
        c.pools, c.pool_count, c.copies, c.copy_count, c.block_tokens = pools, 3, copies, 1, 64
        assert lib.yvx_cuda_kv_pages_copy(C.byref(c), backend.stream, None) == 0, lib.yvx_cuda_last_error_text()
        for x, w in zip(calls, got):
            assert np.array_equal(attend(*x, tables[1]), w)
        outputs.append(got)
    assert all(np.isfinite(x).all() and np.array_equal(x, y) for x, y in zip(*outputs))
