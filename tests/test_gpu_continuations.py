"""Several continuations of one request, as a server runs them: forked requests, beam search and a speculative step."""
import numpy as np
import pytest

from mlcompiler_b200 import capi, synth
from mlcompiler_b200.host import PagePool, PagedAttentionExecutor, PagedKVStorage, RequestKVState

pytestmark = pytest.mark.gpu
P = 64


@pytest.fixture(scope="module")
def model():
    return synth.SyntheticModel(5, 3, 4, 2, 64, 512, 700)


def make_stack(executor, model, capacity=64):
    pool = PagePool(capacity)
    storage = PagedKVStorage(executor, capacity, model.n_layers, P, model.kv_heads, model.head_dim, 2)
    assert storage.initialize()
    ex = PagedAttentionExecutor(executor, model.num_heads, model.kv_heads, model.head_dim, model.n_layers, 0)
    ex.attach_page_pool(pool, P)
    ex.attach_paged_storage(storage)
    assert ex.attach_model(model.to_device())
    return pool, storage, ex


def close(got, want):
    """Two routes through the same kernels: only the order of sums differs (the attention bar of the model tests)."""
    rms = np.sqrt((want.astype(np.float64) ** 2).mean())
    assert np.abs(got - want).max() <= 5e-3 * rms


@pytest.mark.parametrize("prompt", [1, 30, 63, 64, 65, 130])
@pytest.mark.parametrize("reference_order", [False, True])
def test_forked_requests_go_their_own_ways(executor, model, prompt, reference_order):
    pool, storage, ex = make_stack(executor, model)
    ex.set_call_order(reference_order)
    rng = np.random.default_rng(prompt)
    tokens = rng.integers(0, 700, prompt).tolist()
    ex.run_prefill(0, tokens)
    used = pool.pages_in_use()
    assert ex.fork_request(0, 1) and ex.fork_request(0, 2)
    assert pool.pages_in_use() == used
    assert not ex.fork_request(0, 1) and not ex.fork_request(9, 3) and not ex.fork_request(0, 0)
    ways = {r: rng.integers(0, 700, 4).tolist() for r in (0, 1, 2)}
    got = {}
    for i in range(4):
        out = ex.run_decode([(r, ways[r][i], prompt + i) for r in (0, 1, 2)])
        assert all(ok for _, ok, _ in out)
        got = {rid: logits.copy() for rid, _, logits in out}
    tables = [ex.page_state(r)[0] for r in (0, 1, 2)]
    shared = prompt // P
    for t in tables:
        assert t[:shared] == tables[0][:shared]
    assert len({t[shared] for t in tables}) == 3
    for r in (0, 1, 2):
        fresh = 10 + r
        ex.run_prefill(fresh, tokens)
        for i in range(4):
            out = ex.run_decode([(fresh, ways[r][i], prompt + i)])
        close(got[r], out[0][2])
    for r in (0, 1, 2, 10, 11, 12):
        ex.release_request(r)
    assert pool.pages_in_use() == 0


def test_prompt_behind_a_fork(executor, model):
    pool, storage, ex = make_stack(executor, model)
    rng = np.random.default_rng(3)
    head, tail = rng.integers(0, 700, 100).tolist(), rng.integers(0, 700, 50).tolist()
    ex.run_prefill(0, head)
    assert ex.fork_request(0, 1)
    got = ex.run_prefill(1, tail).copy()
    assert ex.page_state(0)[1] == 100 and ex.page_state(1)[1] == 150
    ex.run_prefill(2, head + tail)
    again = ex.run_decode([(1, 5, 150), (2, 5, 150), (0, tail[0], 100)])
    close(again[0][2], again[1][2])
    ex.run_prefill(3, head + tail[:1])
    want = ex.run_prefill(4, head + tail)
    close(got, want)


def test_a_pass_that_runs_out_of_pages_still_owes_no_copy(executor, model):
    """Two pages for the copies of three children: the pass fails, the requests it got to have their own last page, whole."""
    pool, storage, ex = make_stack(executor, model, capacity=3)
    tokens = list(range(20))
    ex.run_prefill(0, tokens)
    for r in (1, 2, 3):
        assert ex.fork_request(0, r)
    out = ex.run_decode([(r, 7, 20) for r in (1, 2, 3)])
    assert not any(ok for _, ok, _ in out)
    ex.release_request(3)
    ex.release_request(0)
    for r in (1, 2):
        assert ex.truncate_request(r, 20)
    out = ex.run_decode([(r, 7, 20) for r in (1, 2)])
    got = [l.copy() for _, ok, l in out if ok]
    assert len(got) == 2
    for r in (1, 2):
        ex.release_request(r)
    ex.run_prefill(5, tokens)
    want = ex.run_decode([(5, 7, 20)])[0][2]
    for g in got:
        close(g, want)


def log_softmax(x):
    x = x.astype(np.float64)
    m = x.max()
    return x - (m + np.log(np.exp(x - m).sum()))


@pytest.mark.parametrize("beams,groups", [(4, 1), (3, 2)])
def test_beam_search(executor, model, beams, groups):
    """Six steps with the selection on the device and shared pages, against a search that recomputes every hypothesis."""
    pool, storage, ex = make_stack(executor, model)
    rng = np.random.default_rng(11)
    prompts = [rng.integers(0, 700, n).tolist() for n in (61, 17)[:groups]]
    n = groups * beams
    for g in range(groups):
        ex.run_prefill(g * beams, prompts[g][:-1])
        for b in range(1, beams):
            assert ex.fork_request(g * beams, g * beams + b)
    texts = [[prompts[g][-1]] for g in range(groups) for _ in range(beams)]
    cum = np.full((groups, beams), -np.inf, np.float32)
    cum[:, 0] = 0.0
    hyps = [[([], 0.0)] for _ in range(groups)]
    for step in range(6):
        slots = [(i, texts[i][-1], len(prompts[i // beams]) - 1 + step) for i in range(n)]
        got = ex.run_decode_beams(slots, beams, cum, beams)
        assert got is not None
        scores, parents, tokens = got
        assert ex.assign_beams(list(range(n)), [g * beams + int(p) for g in range(groups) for p in parents[g]])
        texts = [texts[g * beams + int(parents[g, b])] + [int(tokens[g, b])] for g in range(groups) for b in range(beams)]
        cum = scores.copy()
        for g in range(groups):     # the same step, each hypothesis run on its own from the prompt
            found = []
            for text, score in hyps[g]:
                rid = 1000
                logits = ex.run_prefill(rid, prompts[g] + text)
                ex.release_request(rid)
                lp = log_softmax(logits)
                for t in np.argsort(-lp, kind="stable")[:beams]:
                    found.append((score + lp[t], text + [int(t)]))
            found.sort(key=lambda f: -f[0])
            hyps[g] = [(t, s) for s, t in found[:beams]]
            assert [texts[g * beams + b][1:] for b in range(beams)] == [t for t, _ in hyps[g]]
            assert np.allclose(cum[g], [s for _, s in hyps[g]], atol=0.05)
    for i in range(n):
        ex.release_request(i)
    assert pool.pages_in_use() == 0


def test_beam_refusals(executor, model):
    pool, storage, ex = make_stack(executor, model)
    ex.run_prefill(0, [1, 2, 3])
    assert ex.fork_request(0, 1)
    slots = [(0, 4, 3), (1, 4, 3)]
    cum = np.zeros(2)
    assert ex.run_decode_beams(slots, 3, cum, 2) is None and ex.run_decode_beams(slots, 2, cum[:1], 2) is None
    assert ex.run_decode_beams(slots, 2, cum, 65) is None
    assert ex.run_decode_beams(slots, 2, cum, 2, finished=[0, 1], pad_token=700) is None
    ex.set_call_order(True)
    assert ex.run_decode_beams(slots, 2, cum, 2) is None
    ex.set_call_order(False)
    assert ex.page_state(0)[1] == 3                     # none of them ran
    assert not ex.assign_beams([0, 0], [0, 0]) and not ex.assign_beams([0, 1], [0, 2]) and not ex.assign_beams([0, 9], [0, 0])
    assert not ex.truncate_request(0, 4) and not ex.truncate_request(9, 0)
    assert ex.run_decode_beams(slots, 2, cum, 2) is not None
    s, p, t = ex.run_decode_beams([(0, 4, 4), (1, 4, 4)], 2, cum, 2, finished=[1, 1], pad_token=9)
    assert (t == 9).all() and p[0].tolist() == [0, 1] and (s == 0).all()


@pytest.mark.parametrize("H,KVH,D", [(8, 2, 64), (8, 2, 128), (4, 2, 80)])
@pytest.mark.parametrize("prefix", [10, 60, 200])
def test_speculative_step(H, KVH, D, prefix):
    """Draft, verify, accept: drafted rows are scattered, the tree is verified in one call, the accepted rows move up, the rest
    is forgotten - and the cache and the attention are those of plain decoding along the accepted path."""
    import torch
    ex = capi.Executor(0)
    rng = np.random.default_rng(prefix)
    parents = [-1, -1, 0, 0, 1, 2, 2, 4, 5, 8, 8]       # a tree of 11 drafted tokens
    path = [0, 2, 5, 8, 10]                              # accepted
    n = len(parents)
    capacity = 12
    pool, plain_pool = PagePool(capacity), PagePool(capacity)
    state, plain = RequestKVState(P, 0), RequestKVState(P, 1)
    pool.allocate()                                     # the two caches lie in different pages
    k, v, k2, v2 = (torch.zeros((capacity, P, KVH, D), dtype=torch.float16, device="cuda") for _ in range(4))
    kv = torch.randn((2, prefix + n, KVH, D), device="cuda").half()
    q = torch.randn((n, H, D), device="cuda").half()
    torch.cuda.synchronize()

    def write(st, pl, kp, vp, rows):
        where = [st.extend_one_token(pl) for _ in rows]
        src = torch.tensor(rows, device="cuda")
        a, b = kv[0][src].contiguous(), kv[1][src].contiguous()
        torch.cuda.synchronize()
        ids, slots = [w[0] for w in where], [w[1] for w in where]
        ex.beginForwardPassCB()
        assert ex.encodeScatterKVPairPagedBatched(kp, vp, ids, slots, P, KVH, D, len(rows), a, b, capacity)
        assert ex.flushForwardPassCB()

    write(state, pool, k, v, list(range(prefix + n)))
    tables = (state.page_table, [0, len(state.page_table)])
    o = torch.zeros((n, H, D), dtype=torch.float16, device="cuda")
    pools = ex.pointerArray([k, v])
    kept_off = [0, len(path)]
    torch.cuda.synchronize()
    ex.beginForwardPassCB()
    assert ex.encodePagedTreeAttention(q, k, v, o, *tables, [prefix], [n], ex.treeMask([parents]), 1, H, KVH, D, P, 0.0, capi.MLC_F16,
                                       capi.MLC_F16, capacity), ex.last_error()
    assert ex.encodeCompactKVRows(pools, *tables, [prefix], path, kept_off, 1, P, KVH, D, 2, capacity), ex.last_error()
    assert ex.flushForwardPassCB()
    assert state.truncate(pool, prefix + len(path))
    # plain decoding along the path
    write(plain, plain_pool, k2, v2, list(range(prefix)))
    for i, node in enumerate(path):
        write(plain, plain_pool, k2, v2, [prefix + node])
        one = torch.zeros((1, H, D), dtype=torch.float16, device="cuda")
        table = plain.page_table
        torch.cuda.synchronize()
        assert ex.runPagedFlashAttention(q[node:node + 1].contiguous(), k2, v2, one, table, [0, len(table)], [prefix + i + 1],
                                         [prefix + i], 1, H, KVH, D, P, True, 0.0, capi.MLC_F16, capi.MLC_F16, capacity)
        # both round their weights and their result to fp16: 2^-11 of a mean of |V| each, twice, with |V| below 5
        assert (one[0].float() - o[node].float()).abs().max().item() <= 4 * 2.0**-11 * 5
    total = prefix + len(path)
    assert plain.total_tokens() == state.total_tokens() == total
    for a, b in ((k, k2), (v, v2)):
        for pos in range(total):
            (p0, s0), (p1, s1) = state.locate(pos), plain.locate(pos)
            assert (a[p0, s0] == b[p1, s1]).all()
    ex.close()


def test_ops_in_one_pass_see_one_another(executor):
    """Copy, compaction and tree attention on one stream without a wait in between, then a decode step on the same pools."""
    import torch
    from tests.tree_cases import TreeCase, default_scale, reference
    case = TreeCase(70, [200], [12], 8, 2, 64, mask="chain", slack=8)
    k, v = (torch.from_numpy(x.view(np.int16)).cuda() for x in (case.k, case.v))
    q = torch.from_numpy(case.q).half().cuda()
    o = torch.zeros((case.T, case.H, case.D), dtype=torch.float16, device="cuda")
    free = [p for p in range(case.capacity) if p not in set(case.pt_flat.tolist())]
    other = np.array(free[:4], np.uint32)                # a fork's pages
    pools = executor.pointerArray([k, v])
    torch.cuda.synchronize()
    executor.beginForwardPassCB()
    assert executor.encodeCopyKVPages(pools, case.pt_flat, other, case.P, case.KVH, case.D, 2, case.capacity)
    assert executor.encodePagedTreeAttention(q, k, v, o, other, case.pt_off, case.prefix, case.draft, case.mask, 1, case.H, case.KVH,
                                             case.D, case.P, 0.0, capi.MLC_F16, capi.MLC_F16, case.capacity)
    assert executor.encodeCompactKVRows(pools, other, case.pt_off, [200], [3, 7, 11], [0, 3], 1, case.P, case.KVH, case.D, 2, case.capacity)
    o2 = torch.zeros((1, case.H, case.D), dtype=torch.float16, device="cuda")
    assert executor.encodePagedFlashAttention(q[:1], k, v, o2, other, case.pt_off, [203], [202], 1, case.H, case.KVH, case.D, case.P, True,
                                              0.0, capi.MLC_F16, capi.MLC_F16, case.capacity)
    assert executor.flushForwardPassCB(), executor.last_error()
    qh = q.float().cpu().numpy()
    want, tol = reference(case, qh, default_scale(case), False)
    assert (np.abs(o.float().cpu().numpy() - want) <= tol + 2.0**-11 * np.abs(want) + 2.0**-25).all()
    # what the decode call saw: 200 committed tokens and drafted tokens 3, 7, 11
    case.sees[0][0] = False
    case.sees[0][0, [3, 7, 11]] = True
    want, tol = reference(case, qh, default_scale(case), False)
    assert (np.abs(o2[0].float().cpu().numpy() - want[0]) <= tol[0] + 2.0**-11 * np.abs(want[0]) + 2.0**-25).all()


def small_storage(executor, model):
    """A pool that hands out more pages than the storage holds: a copy into one of those is refused on the host."""
    pool = PagePool(8)
    storage = PagedKVStorage(executor, 3, model.n_layers, P, model.kv_heads, model.head_dim, 2)
    assert storage.initialize()
    ex = PagedAttentionExecutor(executor, model.num_heads, model.kv_heads, model.head_dim, model.n_layers, 0)
    ex.attach_page_pool(pool, P)
    ex.attach_paged_storage(storage)
    assert ex.attach_model(model.to_device())
    return pool, storage, ex


def test_a_pass_whose_copies_fail_leaves_the_shared_page_where_it_was(executor, model):
    pool, storage, ex = small_storage(executor, model)
    tokens = list(range(20))
    ex.run_prefill(0, tokens)
    taken = [pool.allocate(), pool.allocate()]          # the next page is the storage's fourth
    for r in (1, 2):
        assert ex.fork_request(0, r)
    out = ex.run_decode([(r, 7, 20) for r in (1, 2)])
    assert not any(ok for _, ok, _ in out)
    assert [ex.page_state(r)[0] for r in (0, 1, 2)] == [[0]] * 3
    assert pool.owners(0) == 3 and pool.pages_in_use() == 3
    for page in taken:
        assert pool.release(page)
    for r in (1, 2):
        assert ex.truncate_request(r, 20)
    out = ex.run_decode([(r, 7, 20) for r in (1, 2)])
    got = [l.copy() for _, ok, l in out if ok]
    assert len(got) == 2
    for r in (0, 1, 2):
        ex.release_request(r)
    assert pool.pages_in_use() == 0
    ex.run_prefill(5, tokens)
    want = ex.run_decode([(5, 7, 20)])[0][2]
    for g in got:
        close(g, want)


@pytest.mark.parametrize("reference_order", [False, True])
def test_a_prompt_whose_copy_fails_leaves_the_shared_page_where_it_was(executor, model, reference_order):
    pool, storage, ex = small_storage(executor, model)
    ex.set_call_order(reference_order)
    tokens, tail = list(range(20)), list(range(40, 50))
    ex.run_prefill(0, tokens)
    taken = [pool.allocate(), pool.allocate()]
    assert ex.fork_request(0, 1)
    assert len(ex.run_prefill(1, tail)) == 0
    assert ex.page_state(1)[0] == [0] and pool.owners(0) == 2 and pool.pages_in_use() == 3
    for page in taken:
        assert pool.release(page)
    assert ex.truncate_request(1, 20)
    got = ex.run_prefill(1, tail).copy()
    for r in (0, 1):
        ex.release_request(r)
    close(got, ex.run_prefill(5, tokens + tail))
