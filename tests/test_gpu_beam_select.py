"""Beam selection against the definition in 64 bits.

Parents and tokens are whole numbers and must be equal; the inputs keep scores of different beams further apart than the
sums' rounding, or exactly equal. A score is cum + (x - lse): the sum of exponentials is off by the exponential's 2^-21 and
the rounding of short fp32 sums, 2^-20 in all, the score itself is rounded once, 2^-24 of its value."""
import numpy as np
import pytest

from mlcompiler_b200 import capi

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


@pytest.fixture(scope="module")
def ex():
    e = capi.Executor(0)
    yield e
    e.close()


def reference(x, cum, done, n, pad):
    G, B = cum.shape
    V = x.shape[1]
    scores = np.full((G, n), -np.inf)
    parents = np.full((G, n), NONE, np.uint32)
    tokens = np.full((G, n), NONE, np.uint32)
    for g in range(G):
        found = []
        for b in range(B):
            c = float(cum[g, b])
            if done is not None and done[g, b]:
                if c > -np.inf:
                    found.append((-c, b, pad))
                continue
            row = x[g * B + b].astype(np.float64)
            row = np.where(np.isnan(row), -np.inf, row)
            m = row.max()
            if not np.isfinite(m):
                continue
            s = c + (row - (m + np.log(np.exp(row - m).sum())))
            for t in np.lexsort((np.arange(V), -row))[: n]:
                if s[t] > -np.inf:
                    found.append((-s[t], b, int(t)))
        for i, (neg, b, t) in enumerate(sorted(found)[:n]):
            scores[g, i], parents[g, i], tokens[g, i] = -neg, b, t
    return scores, parents, tokens


def in_groups(x, rows):
    V = x.shape[1]
    return np.concatenate([x[:, r: r + rows].reshape(-1) for r in range(0, V, rows)])


def run(ex, x, cum, done=None, n=4, pad=0, rows=0, shift=0, out=None):
    import torch
    G, B = cum.shape
    V = x.shape[1]
    flat = in_groups(x, rows) if rows else x.reshape(-1)
    logits = torch.zeros(flat.size + shift, device="cuda")
    logits[shift:] = torch.from_numpy(flat).cuda()
    c = torch.from_numpy(cum).cuda()
    d = torch.from_numpy(done.astype(np.uint8)).cuda() if done is not None else None
    s = torch.full((G, n), 7.0, device="cuda")
    p, t = (torch.full((G, n), 7, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    ex.beginForwardPassCB()
    ok = ex.encodeBeamSelect(logits.data_ptr() + 4 * shift, c, d, G, B, V, rows, n, pad, s, p, t)
    flushed = ex.flushForwardPassCB()
    assert ok and flushed, ex.last_error()
    return s.cpu().numpy(), p.cpu().numpy().view(np.uint32), t.cpu().numpy().view(np.uint32)


def check(got, want):
    assert (got[1] == want[1]).all() and (got[2] == want[2]).all()
    empty = want[1] == NONE
    assert (got[0][empty] == -np.inf).all()
    s = want[0][~empty]
    assert (np.abs(got[0][~empty] - s) <= 2.0**-20 + 2.0**-24 * np.abs(s)).all()


def make(seed, G, B, V, spread=2.5):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((G * B, V)) * spread).astype(np.float32), (-rng.random((G, B)) * 9).astype(np.float32)


@pytest.mark.parametrize("G,B,V,n", [
    (1, 1, 1, 1), (1, 1, 1, 2), (1, 2, 3, 8), (3, 4, 50, 8), (1, 4, 32000, 8), (2, 5, 32001, 10), (7, 3, 999, 6),
    (1, 64, 300, 64), (5, 1, 8188, 1), (5, 1, 8189, 2), (2, 2, 70001, 64), (40, 4, 5000, 8), (150, 1, 9000, 3), (1, 16, 130000, 32),
])
@pytest.mark.parametrize("done", [False, True])
def test_against_the_definition(ex, G, B, V, n, done):
    x, cum = make(1, G, B, V)
    flags = (np.random.default_rng(2).random((G, B)) < 0.4) if done else None
    check(run(ex, x, cum, flags, n, V // 2), reference(x, cum, flags, n, V // 2))


@pytest.mark.parametrize("rows", [1, 7, 100, 777, 999, 1000, 4000])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_groups_of_vocabulary_rows_and_alignment(ex, rows, shift):
    x, cum = make(3, 2, 3, 1000)
    check(run(ex, x, cum, None, 7, 0, min(rows, 1000), shift), reference(x, cum, None, 7, 0))


@pytest.mark.parametrize("n", [1, 5, 64])
@pytest.mark.parametrize("V", [40, 2000, 40000])
def test_ties_go_to_the_lowest_index(ex, n, V):
    x = np.zeros((6, V), np.float32)
    x[:, ::2] = -0.0                                    # one value
    cum = np.full((2, 3), -1.5, np.float32)
    check(run(ex, x, cum, None, n), reference(x, cum, None, n, 0))
    x[:, 5::7] = 1.0                                    # equal rows, few distinct values
    check(run(ex, x, cum, None, n), reference(x, cum, None, n, 0))


def test_equal_beams(ex):
    x, cum = make(4, 2, 4, 3000)
    x[1:4], x[5:8] = x[0], x[4]
    cum[:] = -2.0
    check(run(ex, x, cum, None, 8), reference(x, cum, None, 8, 0))


def test_first_step_has_one_live_beam(ex):
    x, cum = make(5, 3, 4, 3000)
    cum[:, 1:] = -np.inf
    got = run(ex, x, cum, None, 8)
    check(got, reference(x, cum, None, 8, 0))
    assert (got[1] == 0).all()


@pytest.mark.parametrize("V", [60, 20000])
@pytest.mark.parametrize("left", [0, 1, 3, 40])
def test_masked_logits(ex, V, left):
    x, cum = make(6, 2, 2, V)
    keep = np.random.default_rng(7).choice(V, left, replace=False)
    masked = np.full_like(x, -np.inf)
    masked[:, keep] = x[:, keep]
    check(run(ex, masked, cum, None, 8), reference(masked, cum, None, 8, 0))
    block = np.full_like(x, -np.inf)                    # what is left lies side by side
    block[:, V - left:] = x[:, V - left:] if left else block[:, V:]
    check(run(ex, block, cum, None, 8), reference(block, cum, None, 8, 0))


def test_lowest_value_as_a_mask(ex):
    x, cum = make(8, 1, 2, 500)
    x[:, 3:] = np.finfo(np.float32).min
    check(run(ex, x, cum, None, 3), reference(x, cum, None, 3, 0))


def test_what_is_no_number_is_never_selected(ex):
    x, cum = make(9, 2, 3, 4000)
    x[0, 100:200] = np.nan
    x[1, 17] = np.inf
    x[2] = np.nan
    cum[1, 0] = np.nan
    with np.errstate(invalid="ignore"):
        want = reference(x, cum, None, 6, 0)
    got = run(ex, x, cum, None, 6)
    check(got, want)
    assert (got[1][0] == 0).all() and not (got[1][1] == 0).any()


def test_all_finished(ex):
    x, cum = make(10, 2, 4, 800)
    x[:] = np.nan                                       # not read
    done = np.ones((2, 4), bool)
    got = run(ex, x, cum, done, 6, 9)
    check(got, reference(x, cum, done, 6, 9))
    assert (got[2][:, :4] == 9).all() and (got[1][:, 4:] == NONE).all()


def test_sorted_rows(ex):
    """All the best values lie side by side: many more than n of them pass the threshold."""
    x = np.tile(np.linspace(5, -5, 30000, dtype=np.float32), (4, 1))
    cum = np.array([[0.0, -0.5, -1.0, -1.5]], np.float32)
    check(run(ex, x, cum, None, 64), reference(x, cum, None, 64, 0))
    check(run(ex, x[:, ::-1].copy(), cum, None, 64), reference(x[:, ::-1], cum, None, 64, 0))


def test_large_values(ex):
    x, cum = make(11, 2, 2, 5000)
    check(run(ex, x + 3e4, cum, None, 4), reference(x + np.float32(3e4), cum, None, 4, 0))
    check(run(ex, (x * 1e37).clip(-3e38, 3e38), cum, None, 4), reference((x * 1e37).clip(-3e38, 3e38), cum, None, 4, 0))


def test_replay_and_back_to_back(ex):
    import torch
    sets = []
    for seed, (G, B, V, n) in enumerate([(2, 4, 9000, 8), (30, 2, 400, 3)]):
        x, cum = make(20 + seed, G, B, V)
        dev = [torch.from_numpy(x).cuda(), torch.from_numpy(cum).cuda(), torch.zeros((G, n), device="cuda"),
               torch.zeros((G, n), dtype=torch.int32, device="cuda"), torch.zeros((G, n), dtype=torch.int32, device="cuda")]
        sets.append((x, cum, n, dev, (G, B, V)))
    torch.cuda.synchronize()

    def call(s):
        x, cum, n, d, (G, B, V) = s
        assert ex.encodeBeamSelect(d[0], d[1], None, G, B, V, 0, n, 0, d[2], d[3], d[4]), ex.last_error()

    ex.beginForwardPassCB()
    for _ in range(50):
        for s in sets:
            call(s)
    graphs = []
    for s in sets:
        ex.beginCapture()
        call(s)
        graphs.append(ex.endCapture())
    assert ex.flushForwardPassCB()
    for s in sets:
        for t in s[3][2:]:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for g in graphs:
            g.launch()
    torch.cuda.synchronize()
    for x, cum, n, d, _ in sets:
        check((d[2].cpu().numpy(), d[3].cpu().numpy().view(np.uint32), d[4].cpu().numpy().view(np.uint32)),
              reference(x, cum, None, n, 0))
    for g in graphs:
        g.destroy()


def test_refusals(ex):
    import torch
    x, c = torch.zeros(2, 10, device="cuda"), torch.zeros(1, 2, device="cuda")
    s, p, t = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    done = torch.zeros(2, dtype=torch.uint8, device="cuda")

    def call(x=x, c=c, done=None, G=1, B=2, V=10, rows=0, n=4, pad=0, s=s, p=p, t=t):
        return 0 if ex.encodeBeamSelect(x, c, done, G, B, V, rows, n, pad, s, p, t) else ex.last_status

    assert call() == 2
    ex.beginForwardPassCB()
    assert call() == 0
    assert call(x=None) == 1 and call(c=None) == 1 and call(s=None) == 1 and call(p=None) == 1 and call(t=None) == 1
    assert call(G=0) == 1 and call(B=0) == 1 and call(V=0) == 1 and call(n=0) == 1
    assert call(B=65) == 5 and call(n=65) == 5 and call(V=1 << 31) == 5
    assert call(done=done, pad=10) == 1 and call(done=done, pad=9) == 0 and call(pad=10) == 0
    assert call(s=s.data_ptr() + 1) == 1
    assert ex.flushForwardPassCB()


def test_overlapping_buffers_are_refused(ex):
    import torch
    x, c = torch.zeros(2, 10, device="cuda"), torch.zeros(1, 2, device="cuda")
    done = torch.zeros(8, dtype=torch.uint8, device="cuda")
    s, p, t = (torch.zeros(2, dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32))

    def call(x=x, c=c, done=None, s=s, p=p, t=t):
        return 0 if ex.encodeBeamSelect(x, c, done, 1, 2, 10, 0, 2, 0, s, p, t) else ex.last_status

    ex.beginForwardPassCB()
    assert call(s=c) == 1 and call(t=x) == 1 and call(p=x.data_ptr() + 76) == 1 and call(done=done, p=done) == 1
    assert call(p=t) == 1 and call(s=t.data_ptr() + 4) == 1
    assert call() == 0 and call(done=done) == 0
    assert ex.flushForwardPassCB()


def test_logits_beyond_four_gigabytes(ex):
    """All logits 0 but one of 5 per row, so a row's best score is its cumulated one plus 5 - log(V - 1 + e^5)."""
    import torch
    G, B, V, n = 64, 64, 270001, 5
    x = torch.zeros((G * B, V), device="cuda")
    assert x.numel() * 4 > 1 << 32
    rng = np.random.default_rng(40)
    token = rng.integers(0, V, G * B)
    x[torch.arange(G * B, device="cuda"), torch.from_numpy(token).cuda()] = 5.0
    cum = (rng.permutation(G * B) * 2.0**-9).astype(np.float32).reshape(G, B)   # distinct, and below 8: the next token of a beam is 5 behind
    dev = [torch.from_numpy(cum).cuda(), torch.zeros((G, n), device="cuda")] + [torch.zeros((G, n), dtype=torch.int32, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    ex.beginForwardPassCB()
    assert ex.encodeBeamSelect(x, dev[0], None, G, B, V, 0, n, 0, *dev[1:]), ex.last_error()
    assert ex.flushForwardPassCB(), ex.last_error()
    best = np.argsort(-cum, axis=1, kind="stable")[:, :n]
    assert (dev[2].cpu().numpy() == best).all()
    assert (dev[3].cpu().numpy() == token.reshape(G, B)[np.arange(G)[:, None], best]).all()
    want = np.take_along_axis(cum.astype(np.float64), best, 1) + 5.0 - np.log(V - 1 + np.exp(5.0))
    # The sum's relative error is the logarithm's absolute one. A lane adds up 528 steps in fp32 (2^-24 of the sum each at most, and
    # as much for the 4 additions inside a step); an exponential is off by 2^-22 and by its argument's rounding, 5 * 2^-24; so are the
    # two factors that bring lane and row to one maximum. The score is rounded once.
    tol = (528 + 4 + 3 * 9) * 2.0**-24 + 2.0**-24 * np.abs(want).max()
    assert np.abs(dev[1].cpu().numpy() - want).max() <= tol


def mostly_nan(seed, V, kept):
    """One row of NaN with numbers at `kept` only, in a random order of size."""
    x = np.full(V, np.nan, np.float32)
    x[kept] = np.random.default_rng(seed).permutation(len(kept)) * 0.25 - 3.0
    return x


@pytest.mark.parametrize("n", [1, 2, 4, 8, 40])
@pytest.mark.parametrize("V", [512, 513, 1500, 40000])
def test_rows_of_mostly_nan(ex, n, V):
    """NaN counts as -inf also where it leaves a lane of the first step no number, and where a few numbers are all there is."""
    rng = np.random.default_rng(50)
    rows = [mostly_nan(0, V, np.arange(4)), mostly_nan(1, V, np.arange(V - 5, V)),
            mostly_nan(2, V, np.arange(0, V, 37)), mostly_nan(3, V, np.arange(272, 276))]
    rows += [mostly_nan(4 + i, V, np.flatnonzero(rng.random(V) < 0.2)) for i in range(12)]
    for i, (start, count) in enumerate([(0, 132), (4, 132), (100, 200), (0, 480), (16, 400), (0, 508)]):   # runs of NaN
        x = (rng.standard_normal(V) * 2.5).astype(np.float32)
        x[start: start + count] = np.nan
        rows.append(x)
    x = (rng.standard_normal(V) * 2.5).astype(np.float32)
    x[[0, 1, 2, 3, 128, 129, 130, 131]] = np.nan                 # all that a lane takes for its first part
    rows += [x, np.where(np.arange(V) == 272, 10, np.where(np.arange(V) == 273, 9, x)).astype(np.float32)]
    x = np.stack(rows)
    cum = np.zeros((len(rows), 1), np.float32)
    check(run(ex, x, cum, None, n), reference(x, cum, None, n, 0))
    cum = -np.arange(len(rows), dtype=np.float32).reshape(-1, 2) * 0.015625
    check(run(ex, x, cum, None, n), reference(x, cum, None, n, 0))


def test_small_exponentials_add_up_beside_a_large_one(ex):
    """One likely token per row, the others so far below that a lane's 16 of a step do not reach the last bit of an fp32 sum: over 196
    steps they make 1e-5. (Enough rows that a row is one segment.)"""
    import torch
    G, B, V = 64, 64, 100001
    x = torch.full((G * B, V), -19.5, device="cuda")
    x[:, 0] = 0.0
    cum = -(np.arange(G * B).reshape(G, B) % 64).astype(np.float32)
    dev = [torch.from_numpy(cum).cuda(), torch.zeros((G, 3), device="cuda")] + [torch.zeros((G, 3), dtype=torch.int32, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    ex.beginForwardPassCB()
    assert ex.encodeBeamSelect(x, dev[0], None, G, B, V, 0, 3, 0, *dev[1:]), ex.last_error()
    assert ex.flushForwardPassCB(), ex.last_error()
    scores = np.tile(np.array([0.0, -1.0, -2.0]) - np.log1p((V - 1) * np.exp(-19.5)), (G, 1))
    check([dev[1].cpu().numpy()] + [t.cpu().numpy().view(np.uint32) for t in dev[2:]],
          (scores, np.tile(np.arange(3, dtype=np.uint32), (G, 1)), np.zeros((G, 3), np.uint32)))
