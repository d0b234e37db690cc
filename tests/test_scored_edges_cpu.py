"""Scored attention, the 8-bit cache and page copies at the edges of what they accept, without a GPU."""
import ctypes as C

import pytest

from clori_b200 import abi
from tests.test_scored_cpu import pages_args, scored_problem


def coded_prompt(library, **changes):
    p = scored_problem(kv_code=abi.KV_E4M3, block_table=4096, key_scales=4096, value_scales=4096, block_tokens=64, pool_blocks=1000,
                       query_heads=32, kv_heads=8, key_token_stride=128, value_token_stride=128, key_head_stride=64 * 128,
                       value_head_stride=64 * 128, key_outer_stride=8 * 64 * 128, value_outer_stride=8 * 64 * 128,
                       query_row_stride=32 * 128, query_session_stride=17 * 32 * 128, **changes)
    p.block_table_stride = -(-p.kv_tokens_max // 64)
    library.yvx_cuda_scored_plan(C.byref(p), 148)
    partial = p.sessions * p.query_rows * 32 * p.max_splits * 132 * 4 if p.max_splits > 1 else 0
    return library.yvx_cuda_scored_workspace_bytes(C.byref(p)) - partial


@pytest.mark.parametrize("sessions,tokens,window,most", [
    (64, 32768, 0, 4 << 30), (64, 131072, 0, 4 << 30), (64, 32768, 4096, 64 * 8 * 4288 * 512 + 256), (1, 2000, 0, 8 * 2048 * 512 + 256),
    (3, 1 << 20, 0, 8 * (1 << 20) * 512 + 256), (1, 1 << 20, 1000, 8 * 1152 * 512 + 256), (20000, 1 << 20, 1000, 4 << 30),
])
def test_staged_rows_follow_what_the_call_sees(library, sessions, tokens, window, most):
    staged = coded_prompt(library, sessions=sessions, query_rows=17, kv_tokens_max=tokens, kv_tokens_uniform=tokens, window=window)
    assert 0 < staged <= most


@pytest.mark.parametrize("changes", [
    dict(query_rows=2 ** 29, max_splits=2), dict(sessions=60000, query_rows=5000, max_splits=2), dict(query_rows=2 ** 32 - 1, force_general=1),
    dict(query_rows=2 ** 32 - 1, kv_code=abi.KV_E4M3, block_table=4096, key_scales=4096, value_scales=4096, block_tokens=64,
         block_table_stride=2, pool_blocks=9),
])
def test_calls_beyond_the_grids_are_refused_before_any_launch(library, changes):
    p, n = scored_problem(workspace_bytes=2 ** 64 - 1, **changes), C.c_uint(7)
    assert library.yvx_cuda_scored_attention(C.byref(p), None, C.byref(n)) == abi.YVEX_ERR_BOUNDS and n.value == 0
    assert b"grid" in library.yvx_cuda_last_error_text()


@pytest.mark.parametrize("fields", [
    dict(row_bytes=2 ** 58 + 1), dict(row_bytes=2 ** 60 + 4, segments=2, segment_stride=256),          # rows x row_bytes is 64 again
    dict(segments=2 ** 24 + 1, segment_stride=2 ** 40 - 2 ** 16, block_stride=2 ** 62), dict(segments=2 ** 25 + 1, segment_stride=2 ** 39),
    dict(fixed_bytes=2 ** 41, block_stride=2 ** 42), dict(block_stride=2 ** 61), dict(blocks=2 ** 31 - 1, block_stride=2 ** 40),
])
def test_page_sizes_that_leave_64_bits_are_refused(library, fields):
    a, n = pages_args([], **fields), C.c_uint(5)
    assert library.yvx_cuda_kv_pages_copy(C.byref(a), None, C.byref(n)) == abi.YVEX_ERR_INVALID_ARG and n.value == 0
