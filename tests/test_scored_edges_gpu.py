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
