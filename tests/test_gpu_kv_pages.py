"""Page copies and row compaction inside the paged pools: bit-exact against plain indexing."""
import numpy as np
import pytest

from mlcompiler_b200 import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    e = capi.Executor(0)
    yield e
    e.close()


def make_pools(seed, n, capacity, P, KVH, D, nbytes, offset=0):
    """n pools of random bits (not random numbers: a copy keeps NaN payloads too), each `offset` elements into its allocation."""
    import torch
    rng = np.random.default_rng(seed)
    dt = np.int16 if nbytes == 2 else np.int32
    host = rng.integers(np.iinfo(dt).min, np.iinfo(dt).max, (n, capacity, P, KVH, D), dtype=dt, endpoint=True)
    dev, keep = [], []
    for i in range(n):
        flat = torch.zeros(host[i].size + offset, dtype=torch.int16 if nbytes == 2 else torch.int32, device="cuda")
        flat[offset:] = torch.from_numpy(host[i]).cuda().reshape(-1)
        keep.append(flat)
        dev.append(flat.data_ptr() + offset * nbytes)
    torch.cuda.synchronize()
    return host, keep, capi.Executor.pointerArray(dev)


def now(keep, offset, shape):
    import torch
    torch.cuda.synchronize()
    return np.stack([k[offset:].cpu().numpy().reshape(shape) for k in keep])


@pytest.mark.parametrize("P,KVH,D,nbytes,offset", [
    (64, 4, 64, 2, 0), (64, 8, 128, 2, 0), (64, 2, 128, 4, 0), (7, 3, 5, 2, 0), (1, 1, 1, 2, 0), (16, 2, 20, 2, 0),
    (64, 4, 64, 2, 1), (64, 4, 64, 2, 4), (3, 1, 6, 4, 1),
])
@pytest.mark.parametrize("n_pools", [1, 5])
def test_copy_shapes(ex, P, KVH, D, nbytes, offset, n_pools):
    host, keep, ptrs = make_pools(1, n_pools, 9, P, KVH, D, nbytes, offset)
    src, dst = [3, 3, 8, 5], [0, 7, 1, 5]          # one page to two places; a page to itself
    assert ex.copyKVPages(ptrs, src, dst, P, KVH, D, nbytes, 9), ex.last_error()
    want = host.copy()
    want[:, dst] = host[:, src]
    assert (now(keep, offset, host.shape[1:]) == want).all()


@pytest.mark.parametrize("n_pools,pairs", [(44, 3), (130, 2), (300, 1), (2, 240), (2, 241), (3, 700)])
def test_copy_many_pools_and_pairs(ex, n_pools, pairs):
    host, keep, ptrs = make_pools(2, n_pools, 2 * pairs + 1, 4, 2, 8, 2)
    ids = np.random.default_rng(3).permutation(2 * pairs + 1)
    src, dst = ids[:pairs], ids[pairs: 2 * pairs]
    ex.beginForwardPassCB()
    assert ex.encodeCopyKVPages(ptrs, src, dst, 4, 2, 8, 2, 2 * pairs + 1), ex.last_error()
    assert ex.flushForwardPassCB()
    want = host.copy()
    want[:, dst] = host[:, src]
    assert (now(keep, 0, host.shape[1:]) == want).all()


def test_copy_refusals(ex):
    host, keep, ptrs = make_pools(4, 2, 6, 4, 1, 8, 2)

    def call(src, dst, pools=ptrs, P=4, nbytes=2, cap=6):
        return 0 if ex.copyKVPages(pools, src, dst, P, 1, 8, nbytes, cap) else ex.last_status

    assert call([], []) == 0
    assert call([0, 1], [2]) == 1
    assert call([0], [6]) == 4 and call([6], [0]) == 4 and call([0xFFFFFFFF], [0]) == 4
    assert call([0, 1], [2, 2]) == 1               # one destination, two pairs
    assert call([0, 2], [2, 3]) == 1               # a destination that is a source
    assert call([0, 1], [1, 0]) == 1               # a swap
    assert call([2, 0], [2, 2]) == 0               # a page to itself counts for nothing
    host[:, 2] = host[:, 0]
    assert call([0], [1], P=0) == 1 and call([0], [1], nbytes=3) == 1
    assert call([0], [1], pools=capi.Executor.pointerArray([keep[0], keep[0]])) == 1
    assert call([0], [1], pools=capi.Executor.pointerArray([keep[0], 0])) == 1
    assert call([0], [1], pools=capi.Executor.pointerArray([])) == 1
    assert not ex.encodeCopyKVPages(ptrs, [0], [1], 4, 1, 8, 2, 6) and ex.last_status == 2
    assert (now(keep, 0, host.shape[1:]) == host).all()


def test_copy_checks_against_the_contexts_own_allocations(ex):
    buf = ex.allocateScratchBuffer(5 * 4 * 8 * 2)
    ptrs = capi.Executor.pointerArray([buf])
    assert not ex.copyKVPages(ptrs, [0], [5], 4, 1, 8) and ex.last_status == 4
    assert ex.copyKVPages(ptrs, [0], [4], 4, 1, 8), ex.last_error()
    ex.releaseScratchBuffer(buf)


def compact_reference(host, flat, off, start, kept, P):
    want = host.copy()
    for r, rows in enumerate(kept):
        at = lambda pos: (int(flat[off[r] + pos // P]), pos % P)
        held = [host[:, at(start[r] + k)[0], at(start[r] + k)[1]] for k in rows]
        for i, h in enumerate(held):
            page, slot = at(start[r] + i)
            want[:, page, slot] = h
    return want


@pytest.mark.parametrize("P,KVH,D,nbytes,offset", [(64, 4, 64, 2, 0), (16, 8, 128, 2, 0), (8, 2, 64, 4, 0), (5, 3, 5, 2, 0),
                                                   (1, 1, 8, 2, 0), (64, 4, 64, 2, 3)])
@pytest.mark.parametrize("n_pools", [1, 6])
def test_compact(ex, P, KVH, D, nbytes, offset, n_pools):
    rng = np.random.default_rng(5)
    start = np.array([P - 1, 0, 3 * P + 2, 7], np.uint32)
    kept = [[0, 2, 3, 9, 10, 11, 30], [1], [], sorted(rng.choice(60, 25, replace=False).tolist())]
    need = [-(-(int(s) + (max(k) + 1 if k else 0)) // P) for s, k in zip(start, kept)]
    off = np.concatenate([[0], np.cumsum(need)]).astype(np.uint32)
    capacity = int(off[-1]) + 2
    flat = rng.permutation(capacity)[: off[-1]].astype(np.uint32)
    host, keep, ptrs = make_pools(6, n_pools, capacity, P, KVH, D, nbytes, offset)
    koff = np.concatenate([[0], np.cumsum([len(k) for k in kept])])
    assert ex.compactKVRows(ptrs, flat, off, start, sum(kept, []), koff, 4, P, KVH, D, nbytes, capacity), ex.last_error()
    assert (now(keep, offset, host.shape[1:]) == compact_reference(host, flat, off, start, kept, P)).all()


@pytest.mark.parametrize("batch,n", [(1, 300), (100, 3), (300, 7)])
def test_compact_long_lists(ex, batch, n):
    """Every row moves up by one: each destination is the next move's source."""
    P, KVH, D = 16, 1, 16
    pages = -(-(n + 1) // P)
    rng = np.random.default_rng(7)
    flat = rng.permutation(batch * pages).astype(np.uint32)
    off = (np.arange(batch + 1) * pages).astype(np.uint32)
    host, keep, ptrs = make_pools(8, 3, batch * pages, P, KVH, D, 2)
    kept = [list(range(1, n + 1))] * batch
    ex.beginForwardPassCB()
    assert ex.encodeCompactKVRows(ptrs, flat, off, np.zeros(batch), np.concatenate(kept), np.arange(batch + 1) * n, batch, P, KVH,
                                  D, 2, batch * pages), ex.last_error()
    assert ex.flushForwardPassCB()
    assert (now(keep, 0, host.shape[1:]) == compact_reference(host, flat, off, np.zeros(batch, int), kept, P)).all()


def test_compact_refusals(ex):
    host, keep, ptrs = make_pools(9, 2, 4, 4, 1, 8, 2)
    flat, off = [2, 0, 1], [0, 2, 3]

    def call(start=(2, 0), kept=(1, 3, 1), koff=(0, 2, 3), flat=flat, off=off, cap=4, pools=ptrs, P=4):
        ok = ex.compactKVRows(pools, flat, off, start, kept, koff, len(start), P, 1, 8, 2, cap)
        return 0 if ok else ex.last_status

    assert call(kept=(3, 1, 1)) == 1 and call(kept=(1, 1, 1)) == 1
    assert call(kept=(1, 6, 1)) == 4                                     # position 8 of two pages
    assert call(start=(0xFFFFFFFF, 0)) == 4
    assert call(koff=(0, 3, 2)) == 4 and call(off=(2, 0, 3)) == 4
    assert call(off=(0, 2, 4)) == 1                                      # more pages than the table holds
    assert call(flat=(2, 4, 1)) == 4
    assert call(flat=(2, 0, 2)) == 1                                     # two requests move rows of page 2
    assert call(P=0) == 1
    assert call(pools=capi.Executor.pointerArray([keep[0], keep[0]])) == 1
    assert not ex.encodeCompactKVRows(ptrs, flat, off, (2, 0), (1, 3, 1), (0, 2, 3), 2, 4, 1, 8, 2, 4) and ex.last_status == 2
    assert (now(keep, 0, host.shape[1:]) == host).all()
    assert call(kept=(0, 1, 0)) == 0                                     # nothing moves
    assert (now(keep, 0, host.shape[1:]) == host).all()


def test_pages_and_rows_beyond_four_gigabytes(ex):
    import torch
    P, KVH, D = 64, 8, 128
    capacity = (1 << 32) // (P * KVH * D * 2) + 8
    pool = torch.empty((capacity, P, KVH, D), dtype=torch.int16, device="cuda")
    pool[-8:] = torch.randint(-32768, 32767, (8, P, KVH, D), dtype=torch.int16, device="cuda")
    pool[:2] = 7
    before = pool[-8:].cpu().numpy()
    torch.cuda.synchronize()
    ptrs = capi.Executor.pointerArray([pool.data_ptr()])
    assert ex.copyKVPages(ptrs, [capacity - 1, capacity - 2], [0, capacity - 8], P, KVH, D, 2, capacity), ex.last_error()
    assert ex.compactKVRows(ptrs, [capacity - 4, capacity - 3], [0, 2], [60], [1, 5, 7], [0, 3], 1, P, KVH, D, 2, capacity), ex.last_error()
    torch.cuda.synchronize()
    want = before.copy()
    want[0] = before[6]
    rows = before[4:6].reshape(2 * P, KVH, D)
    moved = rows.copy()
    moved[60:63] = rows[[61, 65, 67]]
    want[4:6] = moved.reshape(2, P, KVH, D)
    assert (pool[-8:].cpu().numpy() == want).all()
    assert (pool[0].cpu().numpy() == before[7]).all() and (pool[1] == 7).all()


def test_a_page_twice_in_one_table_is_refused_where_rows_move(ex):
    host, keep, ptrs = make_pools(9, 1, 4, 4, 2, 8, 2)
    twice = [1, 1, 2]
    assert not ex.compactKVRows(ptrs, twice, [0, 3], [0], [5, 6], [0, 2], 1, 4, 2, 8, 2, 4) and ex.last_status == 1
    assert ex.compactKVRows(ptrs, twice, [0, 3], [8], [1, 2], [0, 2], 1, 4, 2, 8, 2, 4), "only page 2 has moving rows"
    assert ex.compactKVRows(ptrs, twice, [0, 3], [0], [0, 1, 2, 3, 4, 5], [0, 6], 1, 4, 2, 8, 2, 4), "nothing moves"
    want = host.copy()
    want[:, 2, :2] = host[:, 2, 1:3]
    assert (now(keep, 0, host.shape[1:]) == want).all()
