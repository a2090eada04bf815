"""What the branching-generation operators are measured on: attention for a tree of drafted tokens over the paged
cache, copying and compacting pages of that cache, and the selection step of a beam search.

A case is a dict of plain values. `prepare` makes what a caller holds before the call, `run` makes one call (with
`own` the framework's entry points, without it the same result in elementary torch operations), `exact` gives the
result in 64 bits from the operator's definition, `work` the bytes and operations the call cannot do without.
"""
import math
import random

import numpy as np
import torch

own = False

_EXECUTORS = {}


def _executor():
    """One context per device and stream with its pass open, as a serving loop keeps it between flushes. It launches on the stream
    that the tensors are made and read on. (Torch's default stream has the handle 0, for which a context would make a stream of its
    own, ordered with nothing; 1 is CUDA's handle of the same default stream.)"""
    dev, stream = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream or 1
    if (dev, stream) not in _EXECUTORS:
        from mlcompiler_b200 import Executor
        _EXECUTORS[dev, stream] = Executor(dev, stream=stream)
    ex = _EXECUTORS[dev, stream]
    if not ex.hasForwardPassCB():
        ex.beginForwardPassCB()
    return ex


def _checked(ex, ok):
    if not ok:
        raise RuntimeError(ex.last_error())


# ------------------------------------------------------------------------------------------------------- cases
# Head shapes: 32 / 4 / 64 and 32 / 8 / 128 with 64-token pages are the two the decode benchmark runs; 22 and 32
# layers are the depths that go with them, 32000 the vocabulary.
def listed():
    a = {"H": 32, "KVH": 4, "D": 64, "P": 64}
    b = {"H": 32, "KVH": 8, "D": 128, "P": 64}
    return [
        # one user's short chat, a drafted tree of 8 tokens: latency
        {"name": "tree_one_short", "op": "tree", **a, "batch": 1, "ctx": 300, "ctx_hi": 300, "draft": 8, "draft_hi": 8, "dtype": "f16", "mask": "tree"},
        # one user's long document: few rows, all of the GPU has to share one long cache
        {"name": "tree_one_long", "op": "tree", **b, "batch": 1, "ctx": 100001, "ctx_hi": 100001, "draft": 13, "draft_hi": 13, "dtype": "f16", "mask": "tree"},
        # a served batch of ragged contexts and ragged trees
        {"name": "tree_batch32", "op": "tree", **a, "batch": 32, "ctx": 1, "ctx_hi": 4095, "draft": 1, "draft_hi": 26, "dtype": "f16", "mask": "tree"},
        # wide trees over long contexts: the largest
        {"name": "tree_wide_long", "op": "tree", **b, "batch": 16, "ctx": 12000, "ctx_hi": 30000, "draft": 64, "draft_hi": 64, "dtype": "f16", "mask": "tree"},
        # the reference's activation type, fp32 queries and outputs
        {"name": "tree_batch8_f32", "op": "tree", **a, "batch": 8, "ctx": 500, "ctx_hi": 6000, "draft": 5, "draft_hi": 16, "dtype": "f32", "mask": "tree"},
        # a beam search of 4 beams gives each beam its own last page, every layer
        {"name": "copy_beams", "op": "copy", **a, "layers": 22, "capacity": 64, "pairs": 3, "dtype": "f16"},
        # a served batch forks many requests at once (one prompt, many samples)
        {"name": "copy_many", "op": "copy", **b, "layers": 32, "capacity": 256, "pairs": 121, "dtype": "f16"},
        # rows of accepted drafted tokens move up behind the committed ones: one request, then a batch
        {"name": "compact_one", "op": "compact", **a, "layers": 22, "batch": 1, "ctx": 777, "ctx_hi": 777, "draft": 26, "draft_hi": 26, "dtype": "f16"},
        {"name": "compact_batch32", "op": "compact", **b, "layers": 32, "batch": 32, "ctx": 3, "ctx_hi": 400, "draft": 7, "draft_hi": 64, "dtype": "f16"},
        # one beam search of 4 beams over the benchmark's vocabulary: latency
        {"name": "beam_one", "op": "beam", "groups": 1, "beams": 4, "vocab": 32000, "select": 8, "rows": 0, "finished": False},
        # a batch of them on logits in the layout the model step leaves (groups of vocabulary rows)
        {"name": "beam_batch8", "op": "beam", "groups": 8, "beams": 4, "vocab": 32000, "select": 8, "rows": 8000, "finished": True},
        # a large batch over a large vocabulary
        {"name": "beam_large", "op": "beam", "groups": 64, "beams": 8, "vocab": 128000, "select": 16, "rows": 0, "finished": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "copy", "compact", "beam", "beam"])
    if op == "beam":
        beams = _log_int(rng, 1, 16)
        vocab = _log_int(rng, 50, 130000)
        groups = max(1, min(_log_int(rng, 1, 64), 60_000_000 // (beams * vocab)))
        return {"op": op, "groups": groups, "beams": beams, "vocab": vocab, "select": rng.randint(1, 2 * beams),
                "rows": rng.choice([0, 0, max(1, vocab // 4)]), "finished": rng.random() < 0.5}
    D = rng.choice([64, 128])
    KVH = rng.choice([1, 2, 4, 8])
    shape = {"H": KVH * rng.choice([1, 2, 4, 7, 8]), "KVH": KVH, "D": D, "P": rng.choice([16, 32, 64, 64, 64, 128])}
    if op == "copy":
        page = shape["P"] * KVH * D * 2
        layers = rng.choice([1, 16, 22, 32])
        pairs = min(_log_int(rng, 1, 200), max(1, 800_000_000 // (2 * layers * page)))
        return {"op": op, **shape, "layers": layers, "capacity": 2 * pairs + rng.randint(0, 20), "pairs": pairs, "dtype": rng.choice(["f16", "f16", "f32"])}
    batch = _log_int(rng, 1, 48)
    if op == "compact":
        lo = rng.randint(0, 300)
        draft = rng.randint(1, 64)
        return {"op": op, **shape, "layers": rng.choice([1, 16, 22]), "batch": batch, "ctx": lo, "ctx_hi": lo + rng.randint(0, 100),
                "draft": rng.randint(1, draft), "draft_hi": draft, "dtype": "f16"}
    draft = _log_int(rng, 1, 100)
    # bounded by the largest listed case's cache and products
    most = min(400_000_000 // (batch * KVH * D * 4), 100_000_000_000 // (4 * batch * draft * shape["H"] * D), 100_000)
    hi = _log_int(rng, 1, max(2, most))
    return {"op": op, **shape, "batch": batch, "ctx": rng.randint(0, hi), "ctx_hi": hi, "draft": rng.randint(1, draft), "draft_hi": draft,
            "dtype": rng.choice(["f16", "f16", "f32"]), "mask": rng.choice(["tree", "tree", "chain", "bits"])}


def _lengths(case):
    """Committed tokens and drafted tokens of every request: fixed by the case, so that its work is too."""
    r = random.Random("%(op)s %(batch)d %(ctx)d %(ctx_hi)d %(draft)d %(draft_hi)d" % case)
    n = case["batch"]
    return [r.randint(case["ctx"], case["ctx_hi"]) for _ in range(n)], [r.randint(case["draft"], case["draft_hi"]) for _ in range(n)]


def _kept(case, draft):
    """Accepted nodes of a request's tree, as rising indices: the first ones in place, the others from behind."""
    r = random.Random("%d %d %d" % (case["ctx"], case["draft"], draft))
    n = r.randint(1, max(1, min(8, draft // 2)))
    stay = r.randint(0, n - 1)
    moved = sorted(r.sample(range(n, draft), min(n - stay, draft - n)))
    return list(range(stay)) + moved


def work(case):
    op = case["op"]
    if op == "beam":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * case["vocab"] * 4 + rows * 4 + case["groups"] * case["select"] * 12, "flops": 3 * rows * case["vocab"]}
    elem = 4 if case["dtype"] == "f32" else 2
    row = case["KVH"] * case["D"]
    if op == "copy":
        return {"bytes": 2 * case["pairs"] * 2 * case["layers"] * case["P"] * row * elem, "flops": 0}
    ctx, draft = _lengths(case)
    if op == "compact":
        moved = sum(sum(1 for i, k in enumerate(_kept(case, d)) if i != k) for d in draft)
        return {"bytes": max(1, 2 * moved * 2 * case["layers"] * row * elem), "flops": 0}
    tokens = sum(draft)
    kv = sum(c + d for c, d in zip(ctx, draft)) * row * 2 * 2
    return {"bytes": kv + 2 * tokens * case["H"] * case["D"] * elem + tokens * ((case["draft_hi"] + 31) // 32) * 4,
            "flops": 4 * case["H"] * case["D"] * sum(d * (c + 1) for c, d in zip(ctx, draft))}


# ------------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tables(totals, P, rng, slack):
    """Page tables with pages in random order; capacity a little above what is needed."""
    need = [-(-t // P) for t in totals]
    capacity = sum(need) + slack
    ids = rng.permutation(capacity)[: sum(need)].astype(np.uint32)
    off = np.zeros(len(totals) + 1, np.uint32)
    off[1:] = np.cumsum(need)
    return ids, off, capacity


def _tree_inputs(case, seed):
    rng = np.random.default_rng(seed)
    g = _generator(seed)
    H, KVH, D, P = (case[k] for k in ("H", "KVH", "D", "P"))
    ctx, draft = _lengths(case)
    flat, off, capacity = _tables([c + d for c, d in zip(ctx, draft)], P, rng, 3)
    k = torch.randn((capacity, P, KVH, D), generator=g, device="cuda", dtype=torch.float16)
    v = torch.randn((capacity, P, KVH, D), generator=g, device="cuda", dtype=torch.float16)
    for r, (c, d) in enumerate(zip(ctx, draft)):  # slots behind the last token hold whatever was there before
        used = (c + d) % P
        if used:
            k[int(flat[off[r + 1] - 1]), used:] = float("nan")
            v[int(flat[off[r + 1] - 1]), used:] = float("nan")
    dt = torch.float32 if case["dtype"] == "f32" else torch.float16
    q = torch.randn((sum(draft), H, D), generator=g, device="cuda", dtype=torch.float32).to(dt)
    words = (max(draft) + 31) // 32
    masks, sees = [], []
    for d in draft:
        see = np.zeros((d, d), bool)
        for i in range(d):
            if case["mask"] == "bits":
                see[i] = rng.random(d) < 0.3
                continue
            parent = i - 1 if case["mask"] == "chain" else int(rng.integers(max(-1, i - 9), i))
            if parent >= 0:
                see[i] = see[parent]
            see[i, i] = True
        sees.append(see)
        padded = np.zeros((d, words * 32), bool)
        padded[:, :d] = see
        masks.append(np.packbits(padded, axis=1, bitorder="little").view(np.uint32).reshape(d, words))
    return {"case": case, "ctx": ctx, "draft": draft, "flat": flat, "off": off, "capacity": capacity, "k": k, "v": v, "q": q,
            "mask": np.ascontiguousarray(np.concatenate(masks)), "sees": sees}


def _pool_inputs(case, seed):
    rng = np.random.default_rng(seed)
    g = _generator(seed)
    KVH, D, P, L = (case[k] for k in ("KVH", "D", "P", "layers"))
    s = {"case": case}
    if case["op"] == "copy":
        capacity = case["capacity"]
        ids = rng.permutation(capacity).astype(np.uint32)
        s["src"], s["dst"] = rng.choice(ids[case["pairs"]:], case["pairs"]), ids[: case["pairs"]].copy()  # one page may go to several
    else:
        ctx, draft = _lengths(case)
        s["flat"], s["off"], capacity = _tables([c + d for c, d in zip(ctx, draft)], P, rng, 1)
        kept = [_kept(case, d) for d in draft]
        s["start"] = np.array(ctx, np.uint32)
        s["kept"] = np.array(sum(kept, []), np.uint32)
        s["kept_off"] = np.concatenate([[0], np.cumsum([len(k) for k in kept])]).astype(np.uint32)
    s["capacity"] = capacity
    dt = torch.float32 if case["dtype"] == "f32" else torch.float16
    s["pools"] = torch.randn((2 * L, capacity, P, KVH, D), generator=g, device="cuda", dtype=dt)  # K and V of every layer
    return s


def _beam_inputs(case, seed):
    g = _generator(seed)
    G, B, V = case["groups"], case["beams"], case["vocab"]
    logits = torch.randn((G * B, V), generator=g, device="cuda") * 2.5
    logits += 6.0 * torch.randn((G * B, V), generator=g, device="cuda").clamp_(min=2.5).sub_(2.5)  # a few likely tokens
    banned = torch.randint(0, V, (max(1, V // 50),), generator=g, device="cuda")
    logits[:: 3, banned] = float("-inf")  # a grammar or a repetition rule forbids some tokens of some beams
    scores = -torch.rand((G, B), generator=g, device="cuda") * 12.0
    scores = scores.sort(dim=1, descending=True).values.contiguous()
    done = None
    if case["finished"]:
        done = (torch.rand((G, B), generator=g, device="cuda") < 0.25).to(torch.uint8)
    rows = case["rows"] or V
    flat = torch.cat([logits[:, r: r + rows].reshape(-1) for r in range(0, V, rows)])
    return {"case": case, "logits": flat, "scores": scores, "done": done, "pad": 2 % V}


def prepare(case, seed):
    if case["op"] == "tree":
        s = _tree_inputs(case, seed)
        s["out"] = torch.empty_like(s["q"])
        if own:
            ex = _executor()
            s["ex"] = ex
            s["plan"] = ex.createTreePlan(s["flat"], s["off"], s["ctx"], s["draft"], s["mask"], case["batch"], case["H"], case["KVH"],
                                          case["D"], case["P"], s["capacity"])
        else:  # where the rows of every request lie, and who sees whom, as index tensors
            P = case["P"]
            s["at"], s["seen"] = [], []
            for r, (c, d) in enumerate(zip(s["ctx"], s["draft"])):
                pos = np.arange(c + d)
                rows = s["flat"][s["off"][r]: s["off"][r + 1]].astype(np.int64)[pos // P] * P + pos % P
                s["at"].append(torch.from_numpy(rows).cuda())
                s["seen"].append(torch.from_numpy(s["sees"][r]).cuda())
        return s
    if case["op"] == "beam":
        s = _beam_inputs(case, seed)
        n = (case["groups"], case["select"])
        s["out_scores"] = torch.empty(n, device="cuda")
        s["out_parents"] = torch.empty(n, device="cuda", dtype=torch.int32)
        s["out_tokens"] = torch.empty(n, device="cuda", dtype=torch.int32)
        if own:
            s["ex"] = _executor()
        return s
    s = _pool_inputs(case, seed)
    if own:
        s["ex"] = _executor()
        s["pointers"] = s["ex"].pointerArray(list(s["pools"].unbind(0)))
    elif case["op"] == "copy":
        s["src_at"], s["dst_at"] = (torch.from_numpy(s[k].astype(np.int64)).cuda() for k in ("src", "dst"))
    else:
        s["src_at"], s["dst_at"] = (torch.from_numpy(x).cuda() for x in _moves(s, case["P"]))
    return s


def _moves(s, P):
    src, dst = [], []
    for r in range(len(s["start"])):
        table = s["flat"][s["off"][r]: s["off"][r + 1]].astype(np.int64)
        for i, k in enumerate(s["kept"][s["kept_off"][r]: s["kept_off"][r + 1]]):
            a, b = int(s["start"][r]) + int(k), int(s["start"][r]) + i
            src.append(table[a // P] * P + a % P)
            dst.append(table[b // P] * P + b % P)
    return np.array(src, np.int64), np.array(dst, np.int64)


# --------------------------------------------------------------------------------------------------------- run
def run(s):
    case = s["case"]
    if case["op"] == "tree":
        return _run_tree_own(s) if own else _run_tree_plain(s)
    if case["op"] == "beam":
        return _run_beam_own(s) if own else _run_beam_plain(s)
    if case["op"] == "copy":
        if own:
            ex = s["ex"]
            _checked(ex, ex.encodeCopyKVPages(s["pointers"], s["src"], s["dst"], case["P"], case["KVH"], case["D"],
                                              s["pools"].element_size(), s["capacity"]))
        else:
            s["pools"][:, s["dst_at"]] = s["pools"][:, s["src_at"]]
        return s["pools"]
    if own:
        ex = s["ex"]
        _checked(ex, ex.encodeCompactKVRows(s["pointers"], s["flat"], s["off"], s["start"], s["kept"], s["kept_off"], case["batch"],
                                            case["P"], case["KVH"], case["D"], s["pools"].element_size(), s["capacity"]))
    else:
        rows = s["pools"].view(s["pools"].shape[0], -1, case["KVH"] * case["D"])
        rows[:, s["dst_at"]] = rows[:, s["src_at"]]
    return s["pools"]


def _run_tree_own(s):
    from mlcompiler_b200.capi import MLC_F16, MLC_F32
    ex = s["ex"]
    t = MLC_F32 if s["case"]["dtype"] == "f32" else MLC_F16
    _checked(ex, ex.encodePagedTreeAttentionPlanned(s["plan"], s["q"], s["k"], s["v"], s["out"], 0.0, t, t))
    return s["out"]


def _run_tree_plain(s):
    case = s["case"]
    H, KVH, D = case["H"], case["KVH"], case["D"]
    G = H // KVH
    out = s["out"]
    kr, vr = s["k"].view(-1, KVH, D), s["v"].view(-1, KVH, D)
    row = 0
    for c, d, at, seen in zip(s["ctx"], s["draft"], s["at"], s["seen"]):
        k = kr[at].float().permute(1, 2, 0)                                         # [KVH, D, S]
        v = vr[at].float().permute(1, 0, 2)                                         # [KVH, S, D]
        q = s["q"][row: row + d].float().view(d, KVH, G, D).permute(1, 0, 2, 3).reshape(KVH, d * G, D)
        x = (q @ k).mul_(1.0 / math.sqrt(D)).view(KVH, d, G, c + d)
        x[..., c:].masked_fill_(~seen[None, :, None, :], float("-inf"))
        top = x.amax(-1, keepdim=True)
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)        # a row that sees nothing: zeros
        x = x.sub_(top).exp_()
        total = x.sum(-1, keepdim=True).reshape(KVH, d * G, 1)
        o = (x.view(KVH, d * G, c + d) @ v) / torch.where(total == 0, torch.ones_like(total), total)
        out[row: row + d] = o.view(KVH, d, G, D).permute(1, 0, 2, 3).reshape(d, H, D).to(out.dtype)
        row += d
    return out


def _run_beam_own(s):
    case = s["case"]
    ex = s["ex"]
    _checked(ex, ex.encodeBeamSelect(s["logits"], s["scores"], s["done"], case["groups"], case["beams"], case["vocab"], case["rows"],
                                     case["select"], s["pad"], s["out_scores"], s["out_parents"], s["out_tokens"]))
    return [s["out_scores"], s["out_parents"], s["out_tokens"]]


def _run_beam_plain(s):
    case = s["case"]
    G, B, V, n = case["groups"], case["beams"], case["vocab"], case["select"]
    rows = case["rows"] or V
    parts = []
    for r in range(0, V, rows):
        w = min(rows, V - r)
        parts.append(s["logits"][G * B * r: G * B * (r + w)].view(G * B, w))
    x = torch.cat(parts, 1)
    top = x.amax(1, keepdim=True)
    total = (x - top).exp_().sum(1, keepdim=True, dtype=torch.float64)
    # sums of scores are next to one another at the border of the selection: 64 bits
    score = x.double().sub_(top.double() + total.log())
    score += s["scores"].double().view(-1, 1)
    if s["done"] is not None:
        done = s["done"].view(-1).bool()
        score.masked_fill_(done[:, None], float("-inf"))
        score[:, s["pad"]] = torch.where(done, s["scores"].double().view(-1), score[:, s["pad"]])
    score = score.view(G, B * V)
    got, at = [], []
    for g in range(G):  # a stable order: ties go to the lowest index
        v, i = score[g].sort(descending=True, stable=True)
        v, i = v[:n], i[:n]
        if n > B * V:
            v = torch.cat([v, v.new_full((n - B * V,), float("-inf"))])
            i = torch.cat([i, i.new_zeros(n - B * V)])
        got.append(v)
        at.append(i)
    got, at = torch.stack(got), torch.stack(at)
    none = got == float("-inf")
    s["out_scores"].copy_(got)
    s["out_parents"].copy_(torch.where(none, -1, at // V))
    s["out_tokens"].copy_(torch.where(none, -1, at % V))
    return [s["out_scores"], s["out_parents"], s["out_tokens"]]


# ------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    if case["op"] == "tree":
        return _exact_tree(_tree_inputs(case, seed))
    if case["op"] == "beam":
        return _exact_beam(_beam_inputs(case, seed))
    s = _pool_inputs(case, seed)
    pools = s["pools"]
    if case["op"] == "copy":
        before = pools.clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pools[:, b] = before[:, a]
        return pools
    P = case["P"]
    for r in range(case["batch"]):
        table = s["flat"][s["off"][r]: s["off"][r + 1]].tolist()
        places = [int(s["start"][r]) + int(k) for k in s["kept"][s["kept_off"][r]: s["kept_off"][r + 1]]]
        held = [pools[:, table[p // P], p % P].clone() for p in places]
        for i, rows in enumerate(held):
            p = int(s["start"][r]) + i
            pools[:, table[p // P], p % P] = rows
    return pools


def _exact_tree(s):
    """sum over what a drafted token sees of exp(q.k / sqrt(D)) v, over the sum of the weights; by blocks of tokens."""
    case = s["case"]
    H, KVH, D, P = (case[k] for k in ("H", "KVH", "D", "P"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for r, (c, d) in enumerate(zip(s["ctx"], s["draft"])):
        pages = torch.from_numpy(s["flat"][s["off"][r]: s["off"][r + 1]].astype(np.int64)).cuda()
        see = torch.ones((d, c + d), dtype=torch.bool)
        see[:, c:] = torch.from_numpy(s["sees"][r])
        see = see.cuda()
        q = s["q"][first: first + d].double() / math.sqrt(D)
        for h in range(KVH):
            heads = slice(h * (H // KVH), (h + 1) * (H // KVH))
            k = s["k"][pages, :, h].reshape(-1, D)[: c + d].double()
            v = s["v"][pages, :, h].reshape(-1, D)[: c + d].double()
            x = torch.einsum("thd,sd->ths", q[:, heads], k)
            x = torch.where(see[:, None, :], x, torch.full_like(x, float("-inf")))
            w = torch.exp(x - x.amax(2, keepdim=True).clamp(min=-1e300))
            total = w.sum(2, keepdim=True)
            out[first: first + d, heads] = torch.einsum("ths,sd->thd", w, v) / total.clamp(min=1e-300)
        first += d
    return out


def _exact_beam(s):
    case = s["case"]
    G, B, V, n = case["groups"], case["beams"], case["vocab"], case["select"]
    rows = case["rows"] or V
    scores = torch.full((G, n), float("-inf"), dtype=torch.float64)
    parents = torch.full((G, n), -1, dtype=torch.int64)
    tokens = torch.full((G, n), -1, dtype=torch.int64)
    for g in range(G):
        found = []
        for b in range(B):
            m = g * B + b
            cum = float(s["scores"][g, b])
            if s["done"] is not None and int(s["done"][g, b]):
                found.append((-cum, b, s["pad"]))
                continue
            x = torch.cat([s["logits"][G * B * r: G * B * (r + min(rows, V - r))].view(G * B, -1)[m] for r in range(0, V, rows)]).double()
            logp = x - torch.logsumexp(x, 0)
            border = logp.topk(min(n, V)).values[-1]
            for t in (logp >= border).nonzero().view(-1).tolist():
                if float(logp[t]) > float("-inf"):
                    found.append((-(cum + float(logp[t])), b, t))
        for i, (neg, b, t) in enumerate(sorted(found)[:n]):
            scores[g, i], parents[g, i], tokens[g, i] = -neg, b, t
    return [scores, parents, tokens]
