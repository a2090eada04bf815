"""Attention of drafted trees over the paged cache against the definition in 64 bits (tests/tree_cases.py)."""
import numpy as np
import pytest

from mlcompiler_b200 import capi
from tests.tree_cases import TreeCase, default_scale, reference

pytestmark = pytest.mark.gpu

F16, F32 = capi.MLC_F16, capi.MLC_F32


@pytest.fixture(scope="module")
def ex():
    e = capi.Executor(0)
    yield e
    e.close()


class OnDevice:
    def __init__(self, case, q_dtype=F16, o_dtype=F16):
        import torch
        self.q_dtype, self.o_dtype = q_dtype, o_dtype
        self.k, self.v = (torch.from_numpy(x.view(np.int16)).cuda() for x in (case.k, case.v))
        q = torch.from_numpy(case.q)
        self.q = (q if q_dtype == F32 else q.half()).cuda()
        self.q_host = self.q.float().cpu().numpy()
        self.o = torch.full((case.T + 2, case.H, case.D), 77.0, dtype=torch.float32 if o_dtype == F32 else torch.float16, device="cuda")
        torch.cuda.synchronize()

    def result(self, case):
        import torch
        torch.cuda.synchronize()
        got = self.o.float().cpu().numpy()
        assert (got[case.T:] == 77.0).all(), "rows behind the last drafted token were written"
        return got[: case.T]


def check(case, dev, got, scale=None):
    want, tol = reference(case, dev.q_host, scale or default_scale(case), dev.q_dtype == F32 or dev.o_dtype == F32)
    if dev.o_dtype == F16:
        tol = tol + 2.0**-11 * np.abs(want) + 2.0**-25
    assert np.isfinite(got).all()
    err = np.abs(got - want)
    assert (err <= tol).all(), f"error is {(err[tol > 0] / tol[tol > 0]).max():.2f} of its bound"


def run(ex, case, q_dtype=F16, o_dtype=F16, scale=0.0):
    dev = OnDevice(case, q_dtype, o_dtype)
    ok = ex.runPagedTreeAttention(dev.q, dev.k, dev.v, dev.o, *case.tables(), case.N, case.H, case.KVH, case.D, case.P, scale,
                                  q_dtype, o_dtype, case.capacity)
    assert ok, ex.last_error()
    return dev, dev.result(case)


@pytest.mark.parametrize("H,KVH,D,P", [
    (8, 2, 64, 64), (8, 2, 128, 64), (4, 4, 64, 64), (7, 1, 128, 64), (32, 2, 64, 64), (14, 2, 64, 64),
    (8, 2, 64, 16), (8, 2, 128, 32), (8, 2, 128, 128), (4, 2, 64, 192),
    (4, 2, 80, 64), (2, 1, 256, 64), (4, 4, 32, 64), (4, 2, 64, 48), (4, 2, 128, 1), (3, 3, 20, 7),
])
def test_shapes(ex, H, KVH, D, P):
    case = TreeCase(1, [130, 64, 5], [9, 13, 4], H, KVH, D, P)
    check(case, *run(ex, case))


@pytest.mark.parametrize("prefix,draft", [
    ([0], [1]), ([1], [1]), ([63], [1]), ([64], [1]), ([63], [2]), ([0], [64]), ([0], [65]), ([127], [33]),
    ([100, 0, 3], [0, 3, 0]), ([500], [100]), ([640, 64, 1], [64, 1, 31]), ([1000, 2000, 10], [5, 6, 7]),
])
@pytest.mark.parametrize("mask", ["tree", "bits"])
def test_lengths(ex, prefix, draft, mask):
    case = TreeCase(2, prefix, draft, 8, 2, 64, mask=mask)
    check(case, *run(ex, case))
    case = TreeCase(3, prefix, draft, 4, 1, 128, mask=mask)
    check(case, *run(ex, case))


@pytest.mark.parametrize("q_dtype,o_dtype", [(F32, F32), (F32, F16), (F16, F32)])
@pytest.mark.parametrize("D", [64, 128, 96])
def test_types(ex, q_dtype, o_dtype, D):
    case = TreeCase(4, [200, 31, 0], [11, 40, 2], 8, 2, D)
    check(case, *run(ex, case, q_dtype, o_dtype))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("factor", [1e6, 1e-6])
def test_fp32_queries_far_from_one(ex, D, factor):
    case = TreeCase(5, [200], [11], 4, 2, D)
    case.q *= np.float32(factor)
    check(case, *run(ex, case, F32, F32, scale=default_scale(case) / factor), scale=default_scale(case) / factor)


@pytest.mark.parametrize("D", [64, 128, 72])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_that_see_nothing_are_zeros(ex, D, dtype):
    case = TreeCase(6, [0, 0, 3], [5, 70, 2], 4, 2, D, mask="none")
    dev, got = run(ex, case, dtype, dtype)
    assert (got[:75] == 0).all()
    check(case, dev, got)


@pytest.mark.parametrize("D", [64, 128, 72])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_unseen_drafts_have_no_effect_whatever_they_hold(ex, D, dtype, bad):
    """Drafted tokens 2 and 60 hold no numbers; those that see them get none, the others what they would get anyway."""
    case = TreeCase(7, [30, 100], [70, 9], 4, 2, D, mask="tree")
    for i in range(70):      # token 0 is everybody's ancestor; 2 and 60 have no children
        case.sees[0][i, 2] = i == 2
        case.sees[0][i, 60] = i == 60
    for j in (2, 60):
        page, slot = case.where(0, 30 + j)
        case.k[page, slot] = bad
        case.v[page, slot, :, ::3] = bad
    dev, got = run(ex, case, dtype, dtype)
    keep = np.ones(case.T, bool)
    keep[[2, 60]] = False
    for j in (2, 60):        # the reference leaves them out
        case.sees[0][j, j] = False
    want, tol = reference(case, dev.q_host, default_scale(case), dtype == F32)
    if dtype == F16:
        tol = tol + 2.0**-11 * np.abs(want) + 2.0**-25
    assert (np.abs(got - want)[keep] <= tol[keep]).all()
    assert not np.isfinite(got[[2, 60]][:, :, ::3]).any()


@pytest.mark.parametrize("D", [64, 128])
def test_infinite_values_reach_those_that_see_them(ex, D):
    case = TreeCase(8, [70], [9], 4, 2, D, mask="chain")
    page, slot = case.where(0, 70 + 4)
    case.v[page, slot, 1, 5] = np.inf
    _, got = run(ex, case)
    assert np.isfinite(got[:4]).all() and np.isfinite(got[4:, :2]).all()
    assert np.isposinf(got[4:, 2:, 5]).all()
    assert np.isfinite(np.delete(got[4:, 2:], 5, axis=2)).all()


def test_infinite_values_reach_those_that_see_them_when_the_context_is_cut(ex):
    case = TreeCase(9, [9000], [9], 8, 1, 64, mask="chain")
    page, slot = case.where(0, 9004)
    case.v[page, slot, 0, 5] = -np.inf
    _, got = run(ex, case)
    assert np.isfinite(got[:4]).all() and np.isneginf(got[4:, :, 5]).all()
    assert np.isfinite(np.delete(got[4:], 5, axis=2)).all()


def test_large_scores(ex):
    """Scores of some thousands with one sharp maximum at the far end: the running maximum grows all the way."""
    case = TreeCase(10, [300], [6], 4, 2, 64)
    case.q *= 30.0
    check(case, *run(ex, case))


def test_bits_behind_the_drafted_tokens_are_ignored(ex):
    case = TreeCase(11, [77], [5], 4, 2, 64)
    dev = OnDevice(case)
    wide = np.full((5, 3), 0xFFFFFFFF, np.uint32)
    wide[:, 0] = case.mask[:, 0] | np.uint32(0xFFFFFFE0)
    assert ex.runPagedTreeAttention(dev.q, dev.k, dev.v, dev.o, case.pt_flat, case.pt_off, case.prefix, case.draft, wide, case.N,
                                    case.H, case.KVH, case.D, case.P, 0.0, F16, F16, case.capacity), ex.last_error()
    check(case, dev, dev.result(case))


def test_a_chain_is_chunked_prefill(ex):
    """A chain of drafted tokens is what the prefill entry point computes for a chunk."""
    import torch
    case = TreeCase(12, [150, 20], [40, 17], 8, 2, 128, mask="chain")
    dev, got = run(ex, case)
    o = torch.zeros((case.T, case.H, case.D), dtype=torch.float16, device="cuda")
    assert ex.runPagedPrefillAttention(dev.q, dev.k, dev.v, o, case.pt_flat, case.pt_off, case.prefix + case.draft, case.prefix,
                                       case.draft, case.N, case.H, case.KVH, case.D, case.P, 0.0, F16, F16, case.capacity)
    check(case, dev, o.float().cpu().numpy())
    check(case, dev, got)


def plan_for(ex, case):
    return ex.createTreePlan(*case.tables(), case.N, case.H, case.KVH, case.D, case.P, case.capacity)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_plan_and_update(ex, dtype):
    """Several layers on one plan, new tables in between without a wait, a larger and a smaller batch."""
    cases = [TreeCase(20, [300, 20], [9, 3], 8, 2, 64), TreeCase(21, [2500, 7, 0, 64], [20, 33, 1, 64], 8, 2, 64),
             TreeCase(22, [5], [1], 8, 2, 64)]
    devs = [OnDevice(c, dtype, dtype) for c in cases]
    cap = max(c.capacity for c in cases)
    plan = ex.createTreePlan(*cases[0].tables(), cases[0].N, 8, 2, 64, 64, cap)
    ex.beginForwardPassCB()
    for i, (c, d) in enumerate(zip(cases, devs)):
        if i:
            assert plan.update(*c.tables()), ex.last_error()
        for _ in range(2):
            assert ex.encodePagedTreeAttentionPlanned(plan, d.q, d.k, d.v, d.o, 0.0, dtype, dtype), ex.last_error()
    assert ex.flushForwardPassCB(), ex.last_error()
    for c, d in zip(cases, devs):
        check(c, d, d.result(c))
    plan.destroy()


@pytest.mark.parametrize("D", [64, 128])
def test_one_plan_serves_both_types(ex, D):
    """fp16 and fp32 calls, mixed ones too, on one plan without a wait in between."""
    case = TreeCase(23, [3000, 90, 5], [20, 9, 1], 8, 2, D)
    plan = plan_for(ex, case)
    devs = [OnDevice(case, *t) for t in ((F16, F16), (F32, F32), (F16, F32), (F32, F16), (F16, F16))]
    ex.beginForwardPassCB()
    for d in devs:
        assert ex.encodePagedTreeAttentionPlanned(plan, d.q, d.k, d.v, d.o, 0.0, d.q_dtype, d.o_dtype), ex.last_error()
    assert ex.flushForwardPassCB(), ex.last_error()
    for d in devs:
        check(case, d, d.result(case))
    assert ex.lastAttentionKernel() == 4
    plan.destroy()


def test_two_captured_graphs_and_eager_calls_share_the_context(ex):
    a, b = TreeCase(30, [4000, 100], [9, 3], 8, 2, 64), TreeCase(31, [9000], [30], 8, 2, 64)
    da, db = OnDevice(a), OnDevice(b)
    graphs = []
    ex.beginForwardPassCB()
    plans = [plan_for(ex, c) for c in (a, b)]
    for c, d, plan in zip((a, b), (da, db), plans):
        assert ex.encodePagedTreeAttentionPlanned(plan, d.q, d.k, d.v, d.o), ex.last_error()
        assert ex.beginCapture()
        assert ex.encodePagedTreeAttentionPlanned(plan, d.q, d.k, d.v, d.o), ex.last_error()
        graphs.append(ex.endCapture())
    big = TreeCase(32, [20000, 15000], [64, 64], 8, 2, 64)   # grows the scratch after the captures
    dbig = OnDevice(big)
    pbig = plan_for(ex, big)
    assert ex.encodePagedTreeAttentionPlanned(pbig, dbig.q, dbig.k, dbig.v, dbig.o), ex.last_error()
    assert ex.flushForwardPassCB(), ex.last_error()
    first = [d.result(c).copy() for c, d in ((a, da), (b, db))]
    for d in (da, db):
        d.o[: -2].zero_()
    import torch
    torch.cuda.synchronize()
    for _ in range(3):
        for g in graphs:
            g.launch()
    torch.cuda.synchronize()
    for (c, d), before in zip(((a, da), (b, db)), first):
        got = d.result(c)
        check(c, d, got)
        assert (got == before).all(), "a replay does not repeat its results"
    assert not plans[0].update(*a.tables()) and ex.last_status == 5
    for g in graphs:
        g.destroy()


def test_two_contexts_at_once():
    a, b = TreeCase(40, [12000], [9], 8, 2, 64), TreeCase(41, [9000, 9000], [30, 2], 8, 2, 128)
    exs = [capi.Executor(0), capi.Executor(0)]
    devs = [OnDevice(a), OnDevice(b)]
    plans = [plan_for(e, c) for e, c in zip(exs, (a, b))]
    for e in exs:
        e.beginForwardPassCB()
    for _ in range(20):
        for e, d, p in zip(exs, devs, plans):
            assert e.encodePagedTreeAttentionPlanned(p, d.q, d.k, d.v, d.o), e.last_error()
    for e in exs:
        assert e.flushForwardPassCB(), e.last_error()
    for c, d in zip((a, b), devs):
        check(c, d, d.result(c))
    assert not exs[0].beginForwardPassCB() or not exs[0].encodePagedTreeAttentionPlanned(plans[1], devs[1].q, devs[1].k, devs[1].v, devs[1].o)
    assert exs[0].last_status == 1
    for p in plans:
        p.destroy()
    for e in exs:
        e.close()


def test_results_repeat_bit_for_bit(ex):
    case = TreeCase(50, [7000, 300], [26, 8], 32, 4, 64)
    first = run(ex, case)[1]
    for _ in range(3):
        assert (run(ex, case)[1] == first).all()


def test_refusals(ex):
    case = TreeCase(60, [100, 20], [5, 3], 4, 2, 64)
    dev = OnDevice(case)
    flat, off, prefix, draft, mask = case.tables()

    def call(**kw):
        a = dict(q=dev.q, k=dev.k, v=dev.v, o=dev.o, flat=flat, off=off, prefix=prefix, draft=draft, mask=mask, N=2, H=4, KVH=2,
                 D=64, P=64, qd=F16, od=F16, cap=case.capacity)
        a.update(kw)
        ok = ex.runPagedTreeAttention(a["q"], a["k"], a["v"], a["o"], a["flat"], a["off"], a["prefix"], a["draft"], a["mask"],
                                      a["N"], a["H"], a["KVH"], a["D"], a["P"], 0.0, a["qd"], a["od"], a["cap"])
        return 0 if ok else ex.last_status

    assert call() == 0
    assert call(q=None) == 1 and call(k=None) == 1 and call(o=None) == 1
    assert call(qd=2) == 1 and call(od=7) == 1
    assert call(H=5) == 1 and call(KVH=0) == 1 and call(P=0) == 1 and call(D=0) == 1
    assert call(D=260) == 5
    assert call(draft=draft[:1]) == 1 and call(mask=mask[:7]) == 1
    assert call(off=off[::-1].copy()) == 4
    assert call(flat=flat[:-1]) == 1
    assert call(prefix=np.array([124, 20], np.uint32)) == 4      # 129 tokens in two pages
    assert call(prefix=np.array([0xFFFFFFFF, 20], np.uint32)) == 4
    bad = flat.copy()
    bad[1] = case.capacity
    assert call(flat=bad) == 4
    many = np.zeros((43, 1), np.uint32)
    assert call(draft=np.array([40, 3], np.uint32), prefix=np.array([1, 1], np.uint32), mask=many) == 1   # 40 tokens, 32 bits
    assert not ex.hasForwardPassCB()
    assert not ex.encodePagedTreeAttention(dev.q, dev.k, dev.v, dev.o, *case.tables(), 2, 4, 2, 64, 64) and ex.last_status == 2
    with pytest.raises(capi.MlcError):
        ex.createTreePlan(flat, off, prefix, draft[:1], mask, 2, 4, 2, 64, 64)
    with pytest.raises(capi.MlcError):
        ex.createTreePlan(bad, off, prefix, draft, mask, 2, 4, 2, 64, 64, case.capacity)
    plan = plan_for(ex, case)
    assert not ex.encodePagedTreeAttentionPlanned(plan, dev.q, dev.k, dev.v, dev.o) and ex.last_status == 2
    assert not plan.update(bad, off, prefix, draft, mask) and ex.last_status == 4
    ex.beginForwardPassCB()
    assert ex.encodePagedTreeAttentionPlanned(plan, dev.q, dev.k, dev.v, dev.o), "a refused update leaves the plan as it was"
    assert ex.flushForwardPassCB()
    check(case, dev, dev.result(case))
    plan.destroy()


def test_tree_mask_from_parents():
    m = capi.Executor.treeMask([[-1, 0, 0, 2], [], [-1]])
    assert m.shape == (5, 1) and m[:, 0].tolist() == [1, 3, 5, 13, 1]
    assert capi.Executor.treeMask([list(range(-1, 39))]).shape == (40, 2)
    with pytest.raises(ValueError):
        capi.Executor.treeMask([[0]])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_infinite_values_in_every_run_of_a_cta(ex, dtype):
    """More (request, KV head) runs than CTAs: each CTA works through several, every one with an infinite value of its own."""
    rng = np.random.default_rng(70)
    prefix = rng.integers(0, 130, 700)
    case = TreeCase(71, prefix.tolist(), [4] * 700, 2, 2, 64, mask="chain")
    for r in range(case.N):
        page, slot = case.where(r, int(prefix[r]) + 2)
        case.v[page, slot, r % 2, r % 64] = np.inf
    _, got = run(ex, case, dtype, dtype)
    want = np.zeros(got.shape, bool)
    for r in range(case.N):
        want[4 * r + 2: 4 * r + 4, r % 2, r % 64] = True
    assert (np.isposinf(got) == want).all() and np.isfinite(got[~want]).all()


def test_output_over_the_queries_is_refused(ex):
    case = TreeCase(72, [40], [3], 4, 2, 64)
    dev = OnDevice(case)
    plan = plan_for(ex, case)
    ex.beginForwardPassCB()
    assert not ex.encodePagedTreeAttentionPlanned(plan, dev.q, dev.k, dev.v, dev.q) and ex.last_status == 1
    assert not ex.encodePagedTreeAttentionPlanned(plan, dev.q, dev.k, dev.v, dev.q.data_ptr() + 16) and ex.last_status == 1
    assert ex.encodePagedTreeAttentionPlanned(plan, dev.q, dev.k, dev.v, dev.o)
    assert ex.flushForwardPassCB()
    check(case, dev, dev.result(case))
    plan.destroy()


def test_a_plan_goes_while_another_call_is_captured(ex):
    case = TreeCase(73, [700], [9], 8, 2, 64)
    dev = OnDevice(case)
    plan, other = plan_for(ex, case), plan_for(ex, case)
    ex.beginForwardPassCB()
    assert ex.encodePagedTreeAttentionPlanned(plan, dev.q, dev.k, dev.v, dev.o), ex.last_error()
    assert ex.beginCapture()
    other.destroy()
    assert ex.encodePagedTreeAttentionPlanned(plan, dev.q, dev.k, dev.v, dev.o), ex.last_error()
    graph = ex.endCapture()
    assert ex.flushForwardPassCB(), ex.last_error()
    dev.o[: case.T].zero_()
    import torch
    torch.cuda.synchronize()
    graph.launch()
    check(case, dev, dev.result(case))
    graph.destroy()
    plan.destroy()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_more_heads_in_a_group_than_a_row_tile_holds(ex, dtype):
    case = TreeCase(74, [100, 3], [5, 2], 200, 1, 64)
    check(case, *run(ex, case, dtype, dtype))
    case = TreeCase(75, [30], [3], 260, 2, 128)
    check(case, *run(ex, case, dtype, dtype))


@pytest.mark.parametrize("D,KVH", [(64, 8), (80, 8)])
def test_pages_beyond_four_gigabytes(ex, D, KVH):
    """Pools of more than 2^32 bytes, the request's pages at their far end (the rest is left as it is)."""
    import torch
    case = TreeCase(76, [150], [5], 16, KVH, D)
    bytes_per_page = 64 * KVH * D * 2
    capacity = (1 << 32) // bytes_per_page + 1000
    dev = OnDevice(case)
    pools = []
    for host in (case.k, case.v):
        pool = torch.empty((capacity, 64, KVH, D), dtype=torch.float16, device="cuda")
        pool[capacity - case.capacity:] = torch.from_numpy(host).cuda()
        pools.append(pool)
    torch.cuda.synchronize()
    flat, off, prefix, draft, mask = case.tables()
    assert ex.runPagedTreeAttention(dev.q, *pools, dev.o, flat + np.uint32(capacity - case.capacity), off, prefix, draft, mask, 1, 16, KVH, D,
                                    64, 0.0, F16, F16, capacity), ex.last_error()
    assert ex.lastAttentionKernel() == (4 if D == 64 else 1)
    check(case, dev, dev.result(case))


@pytest.mark.parametrize("D", [64, 20])
def test_buffers_off_their_alignment(ex, D):
    """Off 16 bytes is the general kernel's; off an element is refused on the host."""
    import torch
    case = TreeCase(77, [70, 3], [5, 2], 4, 2, D)
    dev = OnDevice(case)
    tables = (*case.tables(), case.N, 4, 2, D, 64, 0.0, F16, F16, case.capacity)
    q, k, v, o = (t.data_ptr() for t in (dev.q, dev.k, dev.v, dev.o))
    for bad in ((q + 1, k, v, o), (q, k + 1, v, o), (q, k, v + 1, o), (q, k, v, o + 1)):
        assert not ex.runPagedTreeAttention(*bad, *tables) and ex.last_status == 1
    shifted = []
    for t in (dev.q, dev.k, dev.v):
        wide = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        wide[1:] = t.reshape(-1)
        shifted.append(wide)
    torch.cuda.synchronize()
    assert ex.runPagedTreeAttention(*(t.data_ptr() + 2 for t in shifted), o, *tables), ex.last_error()
    assert ex.lastAttentionKernel() == 1
    check(case, dev, dev.result(case))


def test_sizes_beyond_the_kernels_types_are_refused(ex):
    case = TreeCase(78, [70], [5], 4, 2, 64)
    dev = OnDevice(case)
    for P, words in (((1 << 32) + 64, None), (1 << 62, None), (1 << 31, None), (64, (1 << 27) + 1)):
        flat, off, prefix, draft, mask = case.tables()
        if words:   # the size alone is looked at
            t = capi.Executor._treeTables(flat, off, prefix, draft, mask, 1)
            args = list(t[1])
            args[-1] = words
            status = ex._lib.mlc_run_paged_tree_attention(ex._h, dev.q.data_ptr(), dev.k.data_ptr(), dev.v.data_ptr(), dev.o.data_ptr(), *args,
                                                          1, 4, 2, 64, P, 0.0, F16, F16, case.capacity)
            assert status == 5
        else:
            assert not ex.runPagedTreeAttention(dev.q, dev.k, dev.v, dev.o, flat, off, prefix, draft, mask, 1, 4, 2, 64, P, 0.0, F16, F16,
                                                case.capacity) and ex.last_status == 5


def test_a_pass_without_any_drafted_token(ex):
    """No request has one: there is nothing to read or write, and empty tensors have no address."""
    import torch
    case = TreeCase(79, [70, 3], [0, 0], 4, 2, 64)
    dev = OnDevice(case)
    empty = torch.zeros((0, 4, 64), dtype=torch.float16, device="cuda")
    assert empty.data_ptr() == 0
    args = (*case.tables(), 2, 4, 2, 64, 64, 0.0, F16, F16, case.capacity)
    assert ex.runPagedTreeAttention(empty, dev.k, dev.v, empty, *args), ex.last_error()
    plan = plan_for(ex, case)
    ex.beginForwardPassCB()
    assert ex.encodePagedTreeAttention(empty, dev.k, dev.v, empty, *args), ex.last_error()
    assert ex.encodePagedTreeAttentionPlanned(plan, empty, dev.k, dev.v, empty), ex.last_error()
    assert not ex.encodePagedTreeAttentionPlanned(plan, empty, None, dev.v, empty) and ex.last_status == 1
    assert ex.flushForwardPassCB()
    dev.result(case)
    plan.destroy()
