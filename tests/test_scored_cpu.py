"""Scored attention, the 8-bit cache and page copies without a GPU: layouts, refusals, host arithmetic, bookkeeping."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import clori_b200
from clori_b200 import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STRUCTS = {"yvx_scored_problem": abi.ScoredProblem, "yvx_kv8_append_args": abi.Kv8AppendArgs,
           "yvx_kv_page_pool": abi.KvPagePool, "yvx_kv_pages_args": abi.KvPagesArgs, "yvex_b200_kv_copy": abi.KvCopy,
           "struct yvx_kv_page_copy": abi.KvCopy, "yvex_b200_kv_pages_pool": abi.KvPagesPool,
           "yvex_b200_attention_scored_request": abi.AttentionScoredRequest,
           "yvex_b200_kv8_append_request": abi.Kv8AppendRequest}


def test_ctypes_mirrors_equal_the_headers(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "yvex_b200/attention.h"', '#include "yvex_b200/cuda_shim.h"',
             'int main(void) {']
    for name, mirror in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {field}));' for field, _ in mirror._fields_]
    source, exe = tmp_path / "probe.c", tmp_path / "probe"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for mirror in STRUCTS.values():
        want += [C.sizeof(mirror)] + [getattr(mirror, field).offset for field, _ in mirror._fields_]
    assert got == want


def scored_problem(**changes):
    p = abi.ScoredProblem()
    p.sessions, p.query_rows, p.query_heads, p.kv_heads, p.head_dim, p.causal, p.scale = 1, 1, 8, 2, 128, 1, 0.1
    p.query_dtype = p.output_dtype = p.kv_dtype = abi.DTYPE_BF16
    p.query = p.output = p.key = p.value = p.status = p.workspace = 4096
    p.query_row_stride = p.query_session_stride = 1024
    p.key_token_stride = p.value_token_stride = 256
    p.key_head_stride = p.value_head_stride = 128
    p.kv_tokens_uniform = p.kv_tokens_max = 100
    p.query_start_from_end, p.chunk_tokens, p.max_splits = 1, 128, 1
    for name, value in changes.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("changes,code", [
    (dict(query=None), abi.YVEX_ERR_INVALID_ARG), (dict(status=None), abi.YVEX_ERR_INVALID_ARG),
    (dict(query_heads=7), abi.YVEX_ERR_INVALID_ARG), (dict(query_rows=0), abi.YVEX_ERR_INVALID_ARG),
    (dict(scale=0.0), abi.YVEX_ERR_INVALID_ARG), (dict(scale=float("inf")), abi.YVEX_ERR_INVALID_ARG),
    (dict(cap=-1.0), abi.YVEX_ERR_INVALID_ARG), (dict(cap=float("nan")), abi.YVEX_ERR_INVALID_ARG),
    (dict(cap=1e-31), abi.YVEX_ERR_INVALID_ARG), (dict(cap=1e-10, scale=1e30), abi.YVEX_ERR_INVALID_ARG),
    (dict(kv_tokens_max=0), abi.YVEX_ERR_INVALID_ARG), (dict(kv_tokens_uniform=101), abi.YVEX_ERR_INVALID_ARG),
    (dict(chunk_tokens=0), abi.YVEX_ERR_INVALID_ARG), (dict(chunk_tokens=100), abi.YVEX_ERR_INVALID_ARG),
    (dict(kv_tokens_max=200, kv_tokens_uniform=200), abi.YVEX_ERR_INVALID_ARG),  # planned for fewer tokens
    (dict(head_dim=257), abi.YVEX_ERR_UNSUPPORTED), (dict(query_dtype=abi.DTYPE_F16), abi.YVEX_ERR_UNSUPPORTED),
    (dict(kv_dtype=abi.DTYPE_I8), abi.YVEX_ERR_UNSUPPORTED), (dict(kv_code=3), abi.YVEX_ERR_UNSUPPORTED),
    (dict(output_dtype=abi.DTYPE_F64), abi.YVEX_ERR_UNSUPPORTED),
    (dict(kv_code=abi.KV_I8), abi.YVEX_ERR_INVALID_ARG),                       # no block table, no scales
    (dict(block_table=4096, block_tokens=64, block_table_stride=1, pool_blocks=9), abi.YVEX_ERR_INVALID_ARG),
    (dict(kv_tokens_max=2 ** 31 - 1000), abi.YVEX_ERR_BOUNDS), (dict(sessions=65536), abi.YVEX_ERR_BOUNDS),
    (dict(max_splits=2, workspace=None), abi.YVEX_ERR_BOUNDS),
    (dict(max_splits=2, workspace=4100, workspace_bytes=1 << 30), abi.YVEX_ERR_BOUNDS),
])
def test_scored_attention_refuses_before_any_launch(library, changes, code):
    p, n = scored_problem(**changes), C.c_uint(7)
    assert library.yvx_cuda_scored_attention(C.byref(p), None, C.byref(n)) == code and n.value == 0


def test_scored_plan_covers_the_tokens_and_is_deterministic(library):
    for rows, tokens, window in [(1, 1, 0), (1, 131072, 0), (8, 70000, 4096), (300, 5000, 0), (4, 4097, 100)]:
        plans = []
        for _ in range(2):
            p = scored_problem(query_rows=rows, kv_tokens_max=tokens, kv_tokens_uniform=tokens, window=window)
            library.yvx_cuda_scored_plan(C.byref(p), 148)
            plans.append((p.chunk_tokens, p.max_splits))
        assert plans[0] == plans[1] and p.chunk_tokens % 64 == 0 and 1 <= p.max_splits <= 8192
        reach = min(window + rows - 1 + 63, tokens + 63) if window else tokens
        assert p.chunk_tokens * p.max_splits >= reach


def append_args(**changes):
    a = abi.Kv8AppendArgs()
    a.sessions, a.tokens, a.kv_heads, a.head_dim, a.code, a.dtype = 1, 1, 2, 128, abi.KV_E4M3, abi.DTYPE_BF16
    a.key = a.value = a.block_table = a.key_codes = a.value_codes = a.key_scales = a.value_scales = a.status = 4096
    a.token_stride = a.session_stride = 256
    a.block_tokens, a.block_table_stride, a.pool_blocks = 64, 4, 8
    a.code_token_stride, a.code_head_stride, a.code_block_stride = 128, 64 * 128, 2 * 64 * 128
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,code", [
    (dict(key=None), abi.YVEX_ERR_INVALID_ARG), (dict(value_scales=None), abi.YVEX_ERR_INVALID_ARG),
    (dict(tokens=0), abi.YVEX_ERR_INVALID_ARG), (dict(code=0), abi.YVEX_ERR_UNSUPPORTED),
    (dict(head_dim=72), abi.YVEX_ERR_UNSUPPORTED), (dict(head_dim=272), abi.YVEX_ERR_UNSUPPORTED),
    (dict(dtype=abi.DTYPE_F16), abi.YVEX_ERR_UNSUPPORTED), (dict(block_tokens=257), abi.YVEX_ERR_UNSUPPORTED),
    (dict(key_codes=4104), abi.YVEX_ERR_INVALID_ARG), (dict(code_token_stride=120), abi.YVEX_ERR_INVALID_ARG),
    (dict(sessions=65536), abi.YVEX_ERR_BOUNDS),
])
def test_kv8_append_refuses_before_any_launch(library, changes, code):
    assert library.yvx_cuda_kv8_append(C.byref(append_args(**changes)), None) == code


def pages_args(copies, blocks=16, **pool_fields):
    pool = abi.KvPagePool(4096, 64 * 256, 0, 256, 0, blocks, 1)
    for name, value in pool_fields.items():
        setattr(pool, name, value)
    a = abi.KvPagesArgs()
    a.pools, a.pool_count, a.block_tokens = C.pointer(pool), 1, 64
    a.copies, a.copy_count = (abi.KvCopy * max(1, len(copies)))(*[abi.KvCopy(1, *c) for c in copies]), len(copies)
    return a


@pytest.mark.parametrize("copies,fields", [
    ([(0, 16, 1)], {}), ([(-1, 3, 1)], {}), ([(1, 2, 65)], {}), ([(3, 3, 4)], {}), ([(0, 1, 4), (2, 1, 4)], {}),
    ([(0, 1, 4), (1, 2, 4)], {}), ([(1, 2, 4), (0, 1, 4)], {}), ([], dict(block_stride=64)), ([], dict(segments=0)),
    ([], dict(segments=2, segment_stride=100)), ([], dict(row_bytes=0)),
])
def test_page_copies_refuse_before_any_launch(library, copies, fields):
    a, n = pages_args(copies, **fields), C.c_uint(5)
    assert library.yvx_cuda_kv_pages_copy(C.byref(a), None, C.byref(n)) == abi.YVEX_ERR_INVALID_ARG and n.value == 0


def test_page_copies_of_nothing_launch_nothing(library):
    a, n = pages_args([]), C.c_uint(5)
    assert library.yvx_cuda_kv_pages_copy(C.byref(a), None, C.byref(n)) == 0 and n.value == 0


def test_row_ranges_equal_a_direct_walk(library):
    rng = np.random.default_rng(2)
    for _ in range(200):
        lengths = rng.integers(0, 9, rng.integers(0, 6)).tolist()
        prefix = rng.integers(0, 12, len(lengths)).tolist() if rng.random() < 0.5 else None
        start, rows = int(rng.integers(0, 10)), int(rng.integers(1, 40))
        first, end = clori_b200.row_ranges(lengths, rows, start, prefix)
        for t in range(rows):
            at, want = 0, (0, 0)
            for d, n in enumerate(lengths):
                if at <= start + t < at + n:
                    seen = min(prefix[d], n) if prefix else 0
                    want = (at, max(start + t + 1, at + seen))
                at += n
            assert (first[t], end[t]) == want
    with pytest.raises(ValueError):
        clori_b200.row_ranges([2 ** 31], 3)
    with pytest.raises(ValueError):
        clori_b200.row_ranges([3], 0)


def test_truncate_frees_blocks_and_keeps_shared_ones(library):
    pool = clori_b200.KvPool(10, 4, 3, 8)
    s = pool.open()
    pool.reserve(s, 18)
    pool.commit(s, 18)
    child = pool.fork(s)
    assert pool.free_blocks() == 5
    pool.truncate(s, 9)
    assert pool.committed(s) == 9 and pool.free_blocks() == 5 and pool.table(s).tolist()[3:] == [-1] * 5
    assert pool.committed(child) == 18 and (pool.table(child)[:5] >= 0).all()
    pool.truncate(child, 0)
    assert pool.free_blocks() == 7 and (pool.table(child) == -1).all()
    with pytest.raises(clori_b200.YvexError):
        pool.truncate(s, 10)
    pool.truncate(s, 8)                       # on a block boundary
    assert pool.free_blocks() == 8
    copy = pool.reserve(s, 3)
    assert copy is None and pool.free_blocks() == 7
    pool.destroy()


def test_compaction_moves_used_blocks_to_the_front_and_keeps_what_sessions_see(library):
    rng = np.random.default_rng(4)
    for trial in range(30):
        blocks, bt = 40, 4
        pool = clori_b200.KvPool(blocks, bt, 8, 12)
        memory = np.full((blocks, bt), -1)
        rows = {}

        def apply(copies):
            was = memory.copy()
            for a, b, n in copies:
                memory[b, :n] = was[a, :n]

        def see(s):
            t = pool.table(s)
            return [int(memory[t[i // bt], i % bt]) for i in range(pool.committed(s))]

        for step in range(60):
            what = rng.integers(0, 5)
            if what == 0 and len(rows) < 8:
                rows[pool.open()] = []
            elif what == 1 and rows and len(rows) < 8:
                parent = int(rng.choice(list(rows)))
                rows[pool.fork(parent)] = list(rows[parent])
            elif what == 2 and rows:
                s = int(rng.choice(list(rows)))
                n = int(rng.integers(1, 9))
                try:
                    copy = pool.reserve(s, n)
                except clori_b200.YvexError:
                    rows[s] = rows[s][:pool.committed(s)]
                    continue
                apply([copy] if copy else [])
                table, at = pool.table(s), len(rows[s])
                for i in range(n):
                    memory[table[(at + i) // bt], (at + i) % bt] = 1000 * step + i
                pool.commit(s, n)
                rows[s] += [1000 * step + i for i in range(n)]
            elif what == 3 and rows:
                s = int(rng.choice(list(rows)))
                keep = int(rng.integers(0, len(rows[s]) + 1))
                pool.truncate(s, keep)
                rows[s] = rows[s][:keep]
            elif what == 4 and rows and rng.random() < 0.5:
                s = int(rng.choice(list(rows)))
                pool.close_session(s)
                del rows[s]
            if rng.random() < 0.2:
                copies = pool.compact()
                sources, targets = [c[0] for c in copies], [c[1] for c in copies]
                assert len(set(sources + targets)) == 2 * len(copies) and all(c[2] == bt for c in copies)
                apply(copies)
                used = blocks - pool.free_blocks()
                memory[used:] = -2
                for s in rows:
                    assert pool.table(s).max(initial=-1) < used
                assert pool.compact() == []
            for s in rows:
                assert see(s) == rows[s]
        pool.destroy()


def test_compaction_with_too_little_room_changes_nothing(library):
    pool = clori_b200.KvPool(8, 4, 2, 8)
    a, b = pool.open(), pool.open()
    for s in (a, b):
        pool.reserve(s, 8)
        pool.commit(s, 8)
    pool.close_session(a)
    before, n = pool.table(b).tolist(), C.c_uint()
    one = (abi.KvCopy * 1)()
    assert library.yvex_b200_kv_pool_compact(pool.handle, one, 1, C.byref(n)) == abi.YVEX_ERR_BOUNDS and n.value == 2
    assert pool.table(b).tolist() == before
    assert library.yvex_b200_kv_pool_compact(None, one, 1, C.byref(n)) == abi.YVEX_ERR_INVALID_ARG
    assert [c[:2] for c in pool.compact()] == [(2, 0), (3, 1)] and pool.table(b).tolist()[:2] == [0, 1]
    pool.destroy()
