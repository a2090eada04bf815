"""The work list of tree attention: every cache tile of every unit in exactly one piece, indices inside their arrays."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "mlcompiler_b200" / "csrc"
NO_SLOT = 0xFFFFFFFF


@pytest.fixture(scope="module")
def work(tmp_path_factory):
    out = tmp_path_factory.mktemp("plan") / "libplan.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", str(CSRC),
                    "-isystem", "/usr/local/cuda/include", str(ROOT / "tests" / "tree_plan_driver.cpp"),
                    str(CSRC / "attn_tree_plan.cpp"), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))

    def run(H, KVH, prefix, draft, max_ctas):
        arr = lambda x: np.ascontiguousarray(x, np.uint32)
        ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)
        prefix, draft = arr(prefix), arr(draft)
        need = [-(-(int(c) + int(d)) // 64) for c, d in zip(prefix, draft)]
        off = arr(np.concatenate([[0], np.cumsum(need)]))
        pieces, splits, row_split, counts = np.zeros(1 << 21, np.uint32), np.zeros(1 << 16, np.uint32), np.zeros(1 << 18, np.uint32), np.zeros(6, np.uint32)
        z = ctypes.c_size_t
        assert lib.tree_work(z(len(prefix)), z(H), z(KVH), ptr(prefix), ptr(draft), ptr(off), ctypes.c_uint32(max_ctas), ptr(pieces),
                             z(pieces.size), ptr(splits), z(splits.size), ptr(row_split), z(row_split.size), ptr(counts))
        n, ctas, ns, rows, slots, slot_rows = counts.tolist()
        return (pieces[: 11 * n].reshape(n, 11).astype(np.int64), splits[: 8 * ns].reshape(ns, 8).astype(np.int64),
                row_split[:rows], ctas, slots, slot_rows, off)

    return run


CASES = [
    (8, 2, [0], [1]), (8, 2, [63], [1]), (8, 2, [64], [1]), (32, 4, [300], [8]), (32, 8, [100001], [13]), (8, 8, [5, 0, 70], [0, 0, 0]),
    (56, 8, [1000] * 48, [100] * 48), (32, 4, list(range(1, 4095, 128)), [1 + i % 26 for i in range(32)]),
    (7, 1, [200000], [100]), (32, 8, [12000, 30000] * 8, [64] * 16), (64, 1, [10, 100000, 1], [1, 64, 3]), (4, 4, [0] * 300, [1] * 300),
]


@pytest.mark.parametrize("H,KVH,prefix,draft", CASES)
@pytest.mark.parametrize("max_ctas", [1, 2, 7, 296])
def test_every_tile_once(work, H, KVH, prefix, draft, max_ctas):
    pieces, splits, row_split, ctas, slots, slot_rows, off = work(H, KVH, prefix, draft, max_ctas)
    G = H // KVH
    assert ctas <= max_ctas and sorted(set(pieces[:, 0])) == list(range(ctas))
    want, token0 = {}, 0
    for r, (c, d) in enumerate(zip(prefix, draft)):
        for h in range(KVH):
            if d:
                want[(token0, h)] = (d * G, -(-(c + d) // 64), c, d, int(off[r]))
        token0 += d
    seen = {}
    for cta, h, row, n_rows, begin, n, slot, c, d, t0, pt in pieces.tolist():
        rows, tiles, c0, d0, pt0 = want[(t0, h)]
        assert (c, d, pt) == (c0, d0, pt0) and 0 < n_rows <= min(128, slot_rows) and row + n_rows <= rows and n > 0
        seen.setdefault((t0, h), {}).setdefault((row, n_rows), []).append((begin, n, slot))
    assert seen.keys() == want.keys()
    used, by_split = [], {(s[3], s[0], s[1]): s for s in splits.tolist()}
    merged = 0
    for unit, tiles_of_rows in seen.items():
        rows, tiles = want[unit][:2]
        at = 0
        for (row, n_rows), parts in sorted(tiles_of_rows.items()):
            assert row == at
            at += n_rows
            pos = 0
            for begin, n, slot in parts:
                assert begin == pos
                pos += n
            assert pos == tiles
            if len(parts) == 1:
                assert parts[0][2] == NO_SLOT and (unit[0], unit[1], row) not in by_split
                continue
            kv_head, r0, nr, t0, first, n_parts, first_row, step = by_split[(unit[0], unit[1], row)]
            assert (nr, n_parts) == (n_rows, len(parts)) and [p[2] for p in parts] == list(range(first, first + n_parts * step, step))
            index = [i for i, s in enumerate(splits.tolist()) if (s[3], s[0], s[1]) == (unit[0], unit[1], row)][0]
            assert (row_split[first_row: first_row + nr] == index).all()
            used += [p[2] for p in parts]
            merged += nr
        assert at == rows
    assert sorted(used) == list(range(slots)) and merged == len(row_split)


def test_row_tiles_of_a_unit_run_side_by_side(work):
    """CTAs of one group have the same runs: what one of them reads from memory, the others find in L2."""
    pieces, *_, ctas, slots, slot_rows, off = work(32, 8, [3000, 900, 4000] * 5, [64, 7, 33] * 5, 296)
    runs = {}
    for cta, h, row, n_rows, begin, n, slot, c, d, t0, pt in pieces.tolist():
        runs.setdefault((t0, h, begin, n), []).append(cta)
    for (t0, h, begin, n), group in runs.items():
        assert max(group) - min(group) == len(group) - 1


def test_runs_are_even(work):
    """A long request beside short ones: no CTA gets much more than its share."""
    pieces, *_, ctas, slots, slot_rows, off = work(32, 8, [100000] + [500] * 31, [16] * 32, 296)
    load = np.zeros(ctas)
    np.add.at(load, pieces[:, 0], pieces[:, 5] + 4)
    assert ctas > 250 and load.max() <= 1.15 * load.sum() / 296 + 8
