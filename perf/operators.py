"""Measured cases of the beam-search operators: selection over beams and vocabulary, and the moves of the decoder states
that follow it (reorder, fork, compact).

A "page" is one decoder row's recurrent state: row p of every plane, a plane being one array of one layer (the fp32 state,
and in bf16 models the bf16 copy that feeds the matrix products).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---- cases --------------------------------------------------------------------------------------------------------

def listed():
    return [
        # selection ------------------------------------------------------------------------------------------------
        # one molecule decoded interactively: the whole cost is latency
        dict(name="select_1x5x51", op="select", n=1, k=5, v=51, ld=64, dtype="fp32", mask="no", keep=True, temp=1.0, done=0.0),
        # a sampling batch of the generate loop (8192 molecules) over the SMILES alphabet, logits in the padded rows that the
        # vocabulary projection writes
        dict(name="select_8192x8x51", op="select", n=8192, k=8, v=51, ld=64, dtype="fp32", mask="no", keep=True, temp=1.0, done=0.3),
        # widest vocabulary of the model, many beams, a grammar mask per beam, sharpened distribution, ranked output
        dict(name="select_1024x32x128", op="select", n=1024, k=32, v=128, ld=128, dtype="bf16", mask="row", keep=False, temp=0.7, done=0.2),
        # a subword vocabulary, few rows: little work per row, long rows, odd width
        dict(name="select_4x8x32001", op="select", n=4, k=8, v=32001, ld=32001, dtype="bf16", mask="vocab", keep=True, temp=1.0, done=0.1),
        # the largest: a batch over a large subword vocabulary
        dict(name="select_64x8x131072", op="select", n=64, k=8, v=131072, ld=131072, dtype="fp32", mask="no", keep=False, temp=1.0, done=0.0),
        # reorder --------------------------------------------------------------------------------------------------
        # one molecule, 3 layers of 512, fp32: latency
        dict(name="reorder_1x5", op="reorder", n=1, k=5, layers=3, width=512, dtype="fp32", pad=0, moved=2),
        # the sampling batch of the default bf16 model, half of the beams moving
        dict(name="reorder_8192x8", op="reorder", n=8192, k=8, layers=3, width=512, dtype="bf16", pad=0, moved=4),
        # an odd width in rows of a wider buffer: no 16-byte row is aligned
        dict(name="reorder_777x7_odd", op="reorder", n=777, k=7, layers=2, width=333, dtype="bf16", pad=5, moved=3),
        # fork -----------------------------------------------------------------------------------------------------
        # start of a search: one latent's state into its beams
        dict(name="fork_1x5", op="fork", n=1, k=5, layers=3, width=512, dtype="fp32", pad=0),
        dict(name="fork_8192x8", op="fork", n=8192, k=8, layers=3, width=512, dtype="bf16", pad=0),
        # compact --------------------------------------------------------------------------------------------------
        # pages of a few beams, some of them done
        dict(name="compact_64", op="compact", n=64, k=8, layers=3, width=512, dtype="bf16", live=0.6),
        # the sampling batch when half of its molecules are done: a page is a molecule's 8 beams
        dict(name="compact_8192", op="compact", n=8192, k=8, layers=3, width=512, dtype="bf16", live=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "fork", "compact"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "select":
        if rng.random() < 0.5:
            v, k = _log(rng, 2, 128), rng.randint(1, 32)
            n = _log(rng, 1, min(16384, 4_000_000 // (k * v)))
        else:
            v, k = _log(rng, 129, 131072), rng.randint(1, 16)
            n = _log(rng, 1, max(1, min(4096, 16_000_000 // (k * v))))
        return dict(op=op, n=n, k=k, v=v, ld=v + rng.choice([0, 0, 1, 13]), dtype=dtype,
                    mask=rng.choice(["no", "vocab", "row"]), keep=rng.random() < 0.5, temp=rng.choice([0.7, 1.0, 1.3]),
                    done=rng.choice([0.0, 0.2, 0.5]))
    layers, width, k = rng.randint(1, 4), _log(rng, 32, 1024), rng.randint(2, 16)
    n = _log(rng, 1, max(1, min(16384, 400_000_000 // (layers * width * k * 6))))
    case = dict(op=op, n=n, k=k, layers=layers, width=width, dtype=dtype)
    if op == "compact":
        return dict(case, live=rng.choice([0.0, 0.3, 0.5, 0.9, 1.0]))
    case["pad"] = rng.choice([0, 0, 3, 8])
    return dict(case, moved=rng.randint(0, k - 1)) if op == "reorder" else case


# ---- inputs -------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _planes(case, pages, width, g):
    """Per layer the fp32 state and, for bf16, the operand copy; each [pages, width], rows `pad` elements wider in memory."""
    out = []
    for _ in range(case["layers"]):
        for t in [torch.float32] + ([torch.bfloat16] if case["dtype"] == "bf16" else []):
            full = torch.empty(pages, width + case.get("pad", 0), device="cuda", dtype=t)
            full.uniform_(-1, 1, generator=g)
            out.append(full[:, :width])
    return out


def prepare(case, seed):
    g = _generator(seed)
    n, k = case["n"], case["k"]
    if case["op"] == "select":
        v = case["v"]
        logits = torch.empty(n, k, case["ld"], device="cuda").normal_(0, 2.5, generator=g).to(TYPES[case["dtype"]])[:, :, :v]
        scores = -40 * torch.rand(n, k, device="cuda", generator=g)
        # a beam that found no continuation, in one place of fifty
        scores[torch.rand(n, k, device="cuda", generator=g) < 0.02] = -math.inf
        finished = torch.rand(n, k, device="cuda", generator=g) < case["done"]
        mask = None
        if case["mask"] != "no":
            mask = torch.rand(*((v,) if case["mask"] == "vocab" else (n, k, v)), device="cuda", generator=g) < 0.75
            mask[..., 1] = True
        if case["mask"] == "row":
            # a grammar that leaves a beam nothing, and garbage where it forbids a symbol
            mask[torch.rand(n, k, device="cuda", generator=g) < 0.02] = False
            logits[~mask & (torch.rand(n, k, v, device="cuda", generator=g) < 0.1)] = math.nan
        return dict(case, logits=logits, scores=scores, finished=finished, mask=mask, eos=v - 2 if v > 2 else 0, pad=v - 1)
    if case["op"] == "reorder":
        # in every group `moved` places take over the state of a place that stays, as equally shared as it can be
        order = torch.rand(n, k, device="cuda", generator=g).argsort(1)
        stay = k - case["moved"]
        parents = torch.arange(k, device="cuda").repeat(n, 1)
        if case["moved"]:
            parents.scatter_(1, order[:, stay:], order[:, torch.arange(case["moved"], device="cuda") % stay])
        return dict(case, planes=_planes(case, n * k, case["width"], g), parents=parents.int())
    if case["op"] == "fork":
        index = torch.arange(n, device="cuda").repeat_interleave(k).int()
        return dict(case, src=_planes(case, n, case["width"], g), dst=_planes(case, n * k, case["width"], g), index=index)
    live = torch.rand(n, device="cuda", generator=g) < case["live"]
    return dict(case, planes=_planes(case, n, k * case["width"], g), live=live)


# ---- one pass -----------------------------------------------------------------------------------------------------

def _plain_select(s):
    logits, scores, finished, eos, pad = s["logits"], s["scores"], s["finished"], s["eos"], s["pad"]
    n, k, v = logits.shape
    # the order of nearly equal candidates hangs on the normaliser: 64 bits
    x = logits.double()
    if s["mask"] is not None:
        x = x.masked_fill(~s["mask"], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = (x - top) / s["temp"]
    logp = (e - e.exp().sum(-1, keepdim=True).log()).float()
    cand = scores[:, :, None] + logp
    alive = torch.isfinite(scores)
    cand = torch.where(torch.isfinite(top) & (alive & ~finished)[:, :, None], cand, -math.inf)
    cand[:, :, pad] = torch.where(alive & finished, scores, cand[:, :, pad])
    cand = cand.flatten(1) + 0.0                      # -0.0 and 0.0 are one score
    # one key: the score's bits in the order of the numbers, then the lower index
    bits = cand.view(torch.int32)
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32) | (k * v - 1 - torch.arange(k * v, device=x.device))
    flat = (k * v - 1) - (key.topk(k, 1).values & 0xFFFFFFFF)
    best = cand.gather(1, flat)
    place = torch.arange(k, device=x.device).expand(n, k)
    found = best > -math.inf
    parent = torch.where(found, flat // v, place)
    token = torch.where(found, flat % v, pad)
    done = ~found | finished.gather(1, parent) | (token == eos)
    if s["keep"]:
        # the best child of a beam stays in its place, the other children take the free places, then what is left
        same = (parent[:, :, None] == parent[:, None, :]) & found[:, None, :]
        first = found & ~same.tril(-1).any(2)
        kept = torch.zeros_like(found).long().scatter_reduce(1, parent, first.long(), "amax")
        free = kept.argsort(dim=1, stable=True)
        nth = torch.where(found & ~first, (found & ~first).long().cumsum(1) - 1, 0)
        rest = (found & ~first).long().sum(1, keepdim=True) + (~found).long().cumsum(1) - 1
        to = torch.where(first, parent, free.gather(1, torch.where(found, nth, rest)))
        best, parent, token, done = (torch.empty_like(t).scatter_(1, to, t) for t in (best, parent, token, done))
        parent = torch.where(best > -math.inf, parent, place)
    return best, parent.int(), token.int(), done


def run(state):
    op = state["op"]
    if own:
        from polygon_amd import vae
        if op == "select":
            return vae.beam_select(state["logits"], state["scores"], state["finished"], mask=state["mask"], temp=state["temp"],
                                   eos=state["eos"], pad=state["pad"], keep_slots=state["keep"])
        if op == "reorder":
            vae.reorder_pages(state["planes"], state["parents"])
            return state["planes"]
        if op == "fork":
            vae.fork_pages(state["dst"], state["src"], state["index"])
            return state["dst"]
        count, where = vae.compact_pages(state["planes"], state["live"])
        return state["planes"] + [count, where]
    if op == "select":
        return _plain_select(state)
    if op == "reorder":
        n, k = state["parents"].shape
        rows = (state["parents"] + torch.arange(n, device="cuda", dtype=torch.int32)[:, None] * k).flatten()
        return [p.copy_(p.index_select(0, rows)) for p in state["planes"]]
    if op == "fork":
        return [d.copy_(s.index_select(0, state["index"])) for d, s in zip(state["dst"], state["src"])]
    live = state["live"]
    pages = torch.arange(live.numel(), device="cuda")
    count = live.sum()
    holes, movers = ~live & (pages < count), live & (pages >= count)
    # the i-th mover goes to the i-th hole; every other page goes to itself
    to_hole = torch.where(holes, holes.cumsum(0) - 1, live.numel())
    from_mover = (~movers).long().argsort(stable=True)           # the movers first, in their order
    hole = (~holes).long().argsort(stable=True)                  # and the holes
    source = torch.where(holes, from_mover[to_hole.clamp(max=live.numel() - 1)], pages)
    where = torch.where(live, torch.where(movers, hole[(movers.cumsum(0) - 1).clamp(min=0)], pages), -1)
    return [p.copy_(p.index_select(0, source)) for p in state["planes"]] + [count.int().reshape(1), where.int()]


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    n, k = case["n"], case["k"]
    if case["op"] == "select":
        # every unfinished beam's logits (and mask) are read once; per logit a scaling, a difference, an exponential (counted
        # as one operation), a sum and two comparisons
        rows, v = n * k * (1 - case["done"]), case["v"]
        mask = {"no": 0, "vocab": v, "row": rows * v}[case["mask"]]
        return {"bytes": rows * v * (2 if case["dtype"] == "bf16" else 4) + mask + 18 * n * k, "flops": 6 * rows * v}
    page = case["layers"] * case["width"] * (6 if case["dtype"] == "bf16" else 4)
    if case["op"] == "reorder":
        read = min(case["moved"], k - case["moved"])
        return {"bytes": n * (read + case["moved"]) * page + 4 * n * k, "flops": n * k}
    if case["op"] == "fork":
        return {"bytes": n * (1 + k) * page + 4 * n * k, "flops": n * k}
    # of the n * live pages that stay, those behind the new end move: a share of (1 - live), read and written
    return {"bytes": n * case["live"] * (1 - case["live"]) * 2 * k * page + 5 * n + 4, "flops": n}


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "select" and case["n"] * case["k"] * case["v"] > 80_000_000:
        return None
    s = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(s)
    if case["op"] == "reorder":
        n, k = case["n"], case["k"]
        old = [p.clone() for p in s["planes"]]
        for j in range(k):
            rows = torch.arange(n, device="cuda") * k
            for p, o in zip(s["planes"], old):
                p[rows + j] = o[rows + s["parents"][:, j].long()]
        return s["planes"]
    if case["op"] == "fork":
        for j in range(case["k"]):
            for d, p in zip(s["dst"], s["src"]):
                d[j::case["k"]] = p
        return s["dst"]
    live = s["live"].cpu().numpy()
    count = int(live.sum())
    where = np.full(case["n"], -1, np.int32)
    where[np.flatnonzero(live)] = np.flatnonzero(live)
    movers, holes = np.flatnonzero(live[count:]) + count, np.flatnonzero(~live[:count])
    where[movers] = holes
    if count and len(holes):
        a, b = torch.from_numpy(holes).cuda(), torch.from_numpy(movers).cuda()
        for p in s["planes"]:
            p[a] = p[b]
    return s["planes"] + [torch.tensor([count], dtype=torch.int32), torch.from_numpy(where)]


def _exact_select(s):
    n, k, v = s["logits"].shape
    scores, finished = s["scores"].cpu().numpy(), s["finished"].cpu().numpy()
    best, parent = np.full((n, k), -np.inf, np.float32), np.tile(np.arange(k, dtype=np.int32), (n, 1))
    token, done = np.full((n, k), s["pad"], np.int32), np.ones((n, k), bool)
    per = max(1, 2_000_000 // (k * v))
    for g0 in range(0, n, per):
        g1 = min(n, g0 + per)
        x = s["logits"][g0:g1].float().cpu().numpy().astype(np.float64)
        if s["mask"] is not None:
            m = s["mask"].cpu().numpy() if s["mask"].dim() == 1 else s["mask"][g0:g1].cpu().numpy()
            x = np.where(m, x, -np.inf)
        with np.errstate(all="ignore"):
            y = x / s["temp"]
            top = y.max(-1, keepdims=True)
            lse = top + np.log(np.exp(y - top).sum(-1, keepdims=True))
            c = scores[g0:g1, :, None] + (y - lse).astype(np.float32)
        c[~np.isfinite(lse[..., 0]) | ~np.isfinite(scores[g0:g1])] = -np.inf
        c[finished[g0:g1]] = -np.inf
        c[..., s["pad"]] = np.where(finished[g0:g1], scores[g0:g1], c[..., s["pad"]])
        for g in range(g0, g1):
            row = c[g - g0].ravel()
            if row.size > 4 * k:
                edge = np.partition(row, -k)[-k]
                near = np.flatnonzero((row >= edge) & (row > -np.inf))
            else:
                near = np.flatnonzero(row > -np.inf)
            near = near[np.argsort(-row[near], kind="stable")][:k]
            entries = [(row[i], i // v, i % v) for i in near]
            taken, places = set(), list(range(len(entries)))
            if s["keep"]:
                for j, (_, p, _) in enumerate(entries):
                    places[j] = None if p in taken else p
                    taken.add(p)
                free = [p for p in range(k) if p not in taken]
                for j, p in enumerate(places):
                    if p is None:
                        places[j] = free.pop(0)
            for j, (c0, p, t) in zip(places, entries):
                best[g, j], parent[g, j], token[g, j] = c0, p, t
                done[g, j] = finished[g, p] or t == s["eos"]
    return best, parent, token, done
