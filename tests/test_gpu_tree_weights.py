"""Tree attention where one token takes nearly all of the weight: the others' weights keep their bits.

Token 0 of every request (a sink) scores `gap` nats above the others and its value is zero, so that the output is made of
the small weights alone. The scores' products are exact here for the sink, and small for the others."""
import numpy as np
import pytest

from mlcompiler_b200 import capi
from tests.tree_cases import TreeCase

pytestmark = pytest.mark.gpu
F16, F32 = capi.MLC_F16, capi.MLC_F32
SCALE = 0.125


@pytest.fixture(scope="module")
def ex():
    e = capi.Executor(0)
    yield e
    e.close()


def sink_case(seed, prefix, draft, H, KVH, D, gap, spread):
    case = TreeCase(seed, prefix, draft, H, KVH, D, mask="chain")
    rng = np.random.default_rng(seed + 100)
    case.q[..., 0] = 4.0
    case.q = case.q.astype(np.float16).astype(np.float32)
    for r in range(case.N):
        for pos in range(int(case.prefix[r]) + int(case.draft[r])):
            page, slot = case.where(r, pos)
            case.k[page, slot] = rng.standard_normal((KVH, D)) * spread
            case.k[page, slot, :, 0] = 0
            case.v[page, slot] += 1                       # the values' mean is not zero
        page, slot = case.where(r, 0)
        case.k[page, slot] = 0
        case.k[page, slot, :, 0] = gap / (4.0 * SCALE)
        case.v[page, slot] = 0
    return case


def reference(case, exact):
    """(O, bound) in 64 bits.

    - a score is off by D * 2^-23 of its sum of magnitudes (the sink's is one exact product); the factor scale * log2(e) and
      the exponent's argument are rounded once each, the second at the size of the gap plus the offset of up to 15
    - an exponential is off by 2^-22; so are the two factors that bring a tile and a run to one reference
    - a weight meets V with 2^-22 of itself in two halves, 2^-11 as one fp16 number, and half a subnormal step of fp16, 2^-25,
      where the largest weight - of its tile of 64 tokens for two halves, of its run for one number - stands at 2^15, or at
      2^8 or more
    - products of a tile are summed in fp32, at worst cut off (64 tokens, 2^-23 each), and so are the tiles; the sum of the
      weights takes 18 additions a tile, rounded
    - the result is rounded once"""
    out, tol = np.zeros((2, case.T, case.H, case.D))
    t, G = 0, case.H // case.KVH
    for r in range(case.N):
        c, d = int(case.prefix[r]), int(case.draft[r])
        places = np.array([case.where(r, p) for p in range(c + d)])
        k, v = (x[places[:, 0], places[:, 1]].astype(np.float64) for x in (case.k, case.v))
        for i in range(d):
            n = c + i + 1                                 # a chain
            tiles = (n + 63) // 64
            for h in range(case.H):
                kh, vh = k[:n, h // G], v[:n, h // G]
                q = case.q[t + i, h].astype(np.float64)
                s = SCALE * (kh @ q)
                w = np.exp(s - s.max())
                total = w.sum()
                o = (w @ vh) / total
                size = SCALE * (np.abs(kh) @ np.abs(q))
                size[0] = 0
                arg = 1.45 * (s.max() - s) + 15
                e = case.D * 2.0**-23 * size + 2.0**-24 * (arg + np.abs(s)) + 3 * 2.0**-22
                mag = (w @ np.abs(vh)) / total
                if exact:
                    top = np.repeat(np.maximum.reduceat(w, np.arange(0, n, 64)), 64)[:n]
                    weight, step = 2.0**-22 * w, 2.0**-40 * top
                else:
                    weight, step = 2.0**-11 * w, np.full(n, 2.0**-33)
                out[t + i, h] = o
                tol[t + i, h] = (((w * e + weight + step) @ np.abs(vh) + (w @ e) * np.abs(o)) / total
                                 + (64 + 16 + tiles) * 2.0**-23 * mag + (18 + tiles) * 2.0**-24 * np.abs(o) + 2.0**-24 * np.abs(o))
        t += d
    return out, tol


def run(ex, case, q_dtype, o_dtype):
    import torch
    k, v = (torch.from_numpy(x.view(np.int16)).cuda() for x in (case.k, case.v))
    q = torch.from_numpy(case.q).cuda()
    q = q if q_dtype == F32 else q.half()
    o = torch.zeros((case.T, case.H, case.D), dtype=torch.float32 if o_dtype == F32 else torch.float16, device="cuda")
    torch.cuda.synchronize()
    assert ex.runPagedTreeAttention(q, k, v, o, *case.tables(), case.N, case.H, case.KVH, case.D, case.P, SCALE, q_dtype, o_dtype,
                                    case.capacity), ex.last_error()
    assert ex.lastAttentionKernel() == 4
    return o.double().cpu().numpy()


def check(ex, case, q_dtype, o_dtype):
    want, tol = reference(case, q_dtype == F32 or o_dtype == F32)
    if o_dtype == F16:
        tol = tol + 2.0**-11 * np.abs(want) + 2.0**-25
    err = np.abs(run(ex, case, q_dtype, o_dtype) - want)
    assert (err <= tol).all(), f"error is {(err / tol).max():.2f} of its bound, {(err / np.abs(want).max()).max():.2e} of the largest value"


@pytest.mark.parametrize("q_dtype,o_dtype", [(F16, F16), (F32, F32), (F32, F16)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("gap", [0, 6, 9, 12, 15, 18])
@pytest.mark.parametrize("spread", [0.0, 0.1])
def test_runs_of_many_tiles_with_a_sink_in_front(ex, q_dtype, o_dtype, D, gap, spread):
    """Enough (request, KV head) runs that none is cut: all of a run has the sink's reference."""
    case = sink_case(1, [600] * 78 + [37, 64], [1] * 80, 4, 4, D, gap, spread)
    check(ex, case, q_dtype, o_dtype)


@pytest.mark.parametrize("q_dtype,o_dtype", [(F16, F16), (F32, F32)])
@pytest.mark.parametrize("gap", [9, 15])
def test_sink_in_a_context_that_is_cut(ex, q_dtype, o_dtype, gap):
    check(ex, sink_case(2, [9000, 150], [2, 5], 8, 2, 64, gap, 0.1), q_dtype, o_dtype)


@pytest.mark.parametrize("q_dtype,o_dtype", [(F16, F16), (F32, F32)])
@pytest.mark.parametrize("D", [64, 128])
def test_references_that_rise_tile_by_tile(ex, q_dtype, o_dtype, D):
    """Every tile's scores lie 3 nats above those of the one before it: the first tiles' weights fade, none outgrows fp16."""
    case = sink_case(3, [600] * 80, [1] * 80, 4, 4, D, 0, 0.1)
    for r in range(case.N):
        for pos in range(1, 601):
            page, slot = case.where(r, pos)
            case.k[page, slot, :, 0] = 3.0 * (pos // 64) / (4.0 * SCALE)
    want, tol = reference(case, q_dtype == F32)
    if o_dtype == F16:
        tol = tol + 2.0**-11 * np.abs(want) + 2.0**-25
    err = np.abs(run(ex, case, q_dtype, o_dtype) - want)
    assert (err <= tol).all(), f"error is {(err / tol).max():.2f} of its bound"
