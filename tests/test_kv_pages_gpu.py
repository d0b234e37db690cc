"""Page copies on a B200: exactly the rows of a copy move, in every pool, and nothing else changes."""
import ctypes as C

import numpy as np
import pytest

import clori_b200
from clori_b200 import abi

pytestmark = pytest.mark.gpu


def expect(pool, copies, page, segments):
    """pool [block, segments * page * lanes] after the copies."""
    blocks = pool.shape[0]
    view = pool.reshape(blocks, segments, page, -1)
    want = view.copy()
    for a, b, n in copies:
        want[b, :, :n] = view[a, :, :n]
    return want.reshape(pool.shape)


@pytest.mark.parametrize("page,lanes,segments,dtype", [(64, 1024, 1, np.uint16), (16, 128, 8, np.int8), (64, 64, 3, np.int8),
                                                       (5, 12, 1, np.int8), (7, 3, 2, np.int8), (64, 33, 1, np.float32)])
@pytest.mark.parametrize("count", [1, 3, 40])
def test_copies_move_their_rows_only(backend, page, lanes, segments, dtype, count):
    rng = np.random.default_rng(page + count)
    blocks = 2 * count + 5
    order = rng.permutation(blocks)
    copies = [(int(order[count + i // 2]), int(order[i]), int(rng.integers(0, page + 1))) for i in range(count)]
    hosts = [rng.integers(0, 127, (blocks, segments * page * lanes)).astype(dtype) for _ in range(3)]
    scales = rng.standard_normal((blocks, 5)).astype(np.float32)
    pools = [backend.tensor("p", h) for h in hosts]
    whole = backend.tensor("s", scales)
    rc, facts = backend.kv_pages_copy([(p, segments) for p in pools] + [(whole, None)], copies, page)
    assert rc == 0 and facts.kernel_launches == 1
    for p, h in zip(pools, hosts):
        assert np.array_equal(p.read(), expect(h, copies, page, segments))
    want = scales.copy()
    for a, b, _ in copies:
        want[b] = scales[a]
    assert np.array_equal(whole.read(), want)


def test_more_copies_and_pools_than_one_launch_holds(backend):
    rng = np.random.default_rng(0)
    count, page, lanes = 1100, 2, 8
    blocks = 2 * count
    order = rng.permutation(blocks)
    copies = [(int(order[count + i]), int(order[i]), page) for i in range(count)]
    hosts = [rng.integers(-99, 99, (blocks, page * lanes)).astype(np.int8) for _ in range(130)]
    pools = [backend.tensor("p", h) for h in hosts]
    rc, facts = backend.kv_pages_copy([(p, 1) for p in pools], copies, page)
    assert rc == 0 and facts.kernel_launches == 6
    for p, h in zip(pools, hosts):
        assert np.array_equal(p.read(), expect(h, copies, page, 1))


def test_empty_lists_and_unneeded_entries(backend):
    host = np.arange(64, dtype=np.int8).reshape(4, 16)
    pool = backend.tensor("p", host)
    assert backend.kv_pages_copy([(pool, 1)], [], 4)[1].kernel_launches == 0
    described = (abi.KvPagesPool * 1)(abi.KvPagesPool(C.cast(pool.ptr, C.c_void_p), 1, 0))
    entries = (abi.KvCopy * 2)(abi.KvCopy(0, 0, 0, 4), abi.KvCopy(1, 1, 2, 3))
    facts, err = abi.OperationFacts(), abi.Error()
    assert backend.lib.yvex_b200_kv_pages_copy_execute(backend.handle, described, 1, entries, 2, 4, C.byref(facts), C.byref(err)) == 0
    assert np.array_equal(pool.read(), expect(host, [(1, 2, 3)], 4, 1))


def test_a_captured_copy_carries_its_lists(backend):
    host = np.arange(6 * 64, dtype=np.uint16).reshape(6, 64)
    pool = backend.tensor("p", host)
    p = abi.KvPagePool(pool.data_ptr, 128, 0, 16, 0, 6, 1)
    copies = (abi.KvCopy * 2)(abi.KvCopy(1, 4, 1, 8), abi.KvCopy(1, 5, 0, 3))
    a = abi.KvPagesArgs()
    a.pools, a.pool_count, a.copies, a.copy_count, a.block_tokens = C.pointer(p), 1, copies, 2, 8
    lib, graph = backend.lib, C.c_void_p()
    assert lib.yvx_cuda_graph_capture_begin(backend.stream) == 0
    assert lib.yvx_cuda_kv_pages_copy(C.byref(a), backend.stream, None) == 0
    assert lib.yvx_cuda_graph_capture_end(backend.stream, C.byref(graph)) == 0
    copies[0].source_block, copies[1].destination_block = 3, 3      # the lists were read when the call was made
    p.base = None
    for _ in range(2):
        pool.write(host)
        assert lib.yvx_cuda_graph_launch(graph, backend.stream) == 0
        assert lib.yvx_cuda_stream_synchronize(backend.stream) == 0
        assert np.array_equal(pool.read(), expect(host, [(4, 1, 8), (5, 0, 3)], 8, 1))
    lib.yvx_cuda_graph_destroy(graph)


def test_operator_refusals(backend):
    pool = backend.tensor("p", np.zeros((4, 64), np.int8))
    call = lambda pools, copies, page: backend.kv_pages_copy(pools, copies, page, check=False)[0]
    assert call([(pool, 1)], [(0, 1, 8)], 8) == 0
    assert call([], [(0, 1, 8)], 8) == abi.YVEX_ERR_INVALID_ARG
    assert call([(pool, 1)], [(0, 1, 8)], 0) == abi.YVEX_ERR_INVALID_ARG
    assert call([(pool, 1)], [(0, 1, 8), (1, 2, 8)], 8) == abi.YVEX_ERR_INVALID_ARG
    assert call([(pool, 1)], [(0, 4, 8)], 8) == abi.YVEX_ERR_INVALID_ARG
    assert call([(pool, 3)], [(0, 1, 8)], 8) == abi.YVEX_ERR_FORMAT
    with clori_b200.Backend(0) as other:
        assert call([(other.tensor("p", np.zeros((4, 64), np.int8)), 1)], [(0, 1, 8)], 8) == abi.YVEX_ERR_FORMAT
