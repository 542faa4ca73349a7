"""Selection over beams and vocabulary, and the moves of decoder state pages, against plain 64-bit (numpy) statements of their
definitions.  Whole numbers must be equal; pages are copies and must be equal bit for bit."""
import numpy as np
import pytest
import torch

from polygon_amd import vae
from polygon_amd._lib import PolygonHipError

pytestmark = pytest.mark.gpu
INF = float("inf")


def ref_select(logits, scores, finished=None, mask=None, temp=1.0, eos=-1, pad=0, keep_slots=False):
    x = logits.detach().cpu().double().numpy()
    s = scores.cpu().numpy()
    n, K, V = x.shape
    fin = np.zeros((n, K), bool) if finished is None else finished.cpu().numpy().astype(bool)
    ok = np.ones((n, K, V), bool) if mask is None else np.broadcast_to(mask.cpu().numpy().astype(bool), (n, K, V))
    out = [np.full((n, K), -np.inf, np.float32), np.tile(np.arange(K, dtype=np.int32), (n, 1)), np.full((n, K), pad, np.int32),
           np.ones((n, K), bool)]
    for g in range(n):
        cand = []
        for k in range(K):
            if not np.isfinite(s[g, k]):
                continue
            if fin[g, k]:
                cand.append((-s[g, k], k * V + pad))
                continue
            allowed = np.flatnonzero(ok[g, k])
            y = x[g, k, allowed]
            if y.size == 0 or np.isnan(y).any() or not np.isfinite(y.max()):
                continue
            e = (y - y.max()) / temp
            with np.errstate(over="ignore"):
                c = s[g, k] + (e - np.log(np.exp(e).sum())).astype(np.float32)
            best = np.lexsort((allowed, -c))[:K]
            cand += [(-c[i], k * V + allowed[i]) for i in best if c[i] > -np.inf]
        cand.sort()
        taken, place = set(), []
        for c, f in cand[:K]:
            p = f // V
            place.append(p if keep_slots and p not in taken else None)
            taken.add(p)
        free = [p for p in range(K) if p not in taken] if keep_slots else []
        for j, (c, f) in enumerate(cand[:K]):
            p = j if not keep_slots else place[j] if place[j] is not None else free.pop(0)
            out[0][g, p], out[1][g, p], out[2][g, p] = -c, f // V, f % V
            out[3][g, p] = fin[g, f // V] or f % V == eos
    return out


def check_select(logits, scores, **kw):
    got = vae.beam_select(logits, scores, **kw)
    want = ref_select(logits, scores, **kw)
    for name, a, b in zip(got._fields[1:], got[1:], want[1:]):
        assert np.array_equal(a.cpu().numpy(), b), name
    a, b = got.scores.cpu().numpy(), want[0]
    assert np.array_equal(np.isfinite(a), np.isfinite(b))
    f = np.isfinite(b)
    # both round the log-probability and the sum once: at most one step apart where the 64-bit values straddle a rounding edge
    lim = 2.0 ** -23 * (2 * np.abs(b[f]) + np.abs(scores.cpu().numpy()[np.isfinite(scores.cpu().numpy())]).max(initial=0.0))
    assert (np.abs(a[f] - b[f]) <= lim).all()
    return got


def make(n, K, V, dtype=torch.float32, seed=0, dead=0.1, done=0.2):
    g = torch.Generator().manual_seed(seed * 1000 + n + K + V)
    logits = (torch.randn(n, K, V, generator=g) * 2.5).to(dtype).cuda()
    scores = -20 * torch.rand(n, K, generator=g)
    scores[torch.rand(n, K, generator=g) < dead] = -INF
    return logits, scores.cuda(), (torch.rand(n, K, generator=g) < done).cuda()


SHAPES = [(1, 1, 1), (3, 2, 1), (5, 1, 7), (2, 32, 2), (4, 5, 3), (1, 5, 51), (130, 8, 51), (9, 8, 64), (9, 8, 65), (33, 32, 128),
          (17, 31, 127), (3, 7, 129), (5, 16, 257), (2, 32, 512), (3, 4, 1000), (2, 8, 1025), (2, 16, 5003), (1, 3, 40001),
          (3, 32, 9000), (1, 16, 70000)]


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,K,V", SHAPES)
def test_select(n, K, V, dt, keep):
    logits, scores, fin = make(n, K, V, dt)
    check_select(logits, scores, finished=fin, eos=V - 1, pad=V // 2, keep_slots=keep)
    check_select(logits, scores, temp=0.6, keep_slots=keep)


@pytest.mark.parametrize("V", [51, 128, 700, 3001])
@pytest.mark.parametrize("kind", ["vocab", "beam", "group", "row"])
def test_select_mask(V, kind):
    n, K = 7, 6
    logits, scores, fin = make(n, K, V, torch.float32, seed=1)
    shape = dict(vocab=(V,), beam=(K, V), group=(n, 1, V), row=(n, K, V))[kind]
    mask = torch.rand(shape, generator=torch.Generator().manual_seed(V)).cuda() < 0.5
    if kind == "row":
        mask[2] = False                  # a group nothing is left to
        mask[3, 1] = False               # a beam nothing is left to
        mask[4] = False
        mask[4, :, 3] = True             # one symbol each
    # what the mask forbids may hold anything
    junk = torch.tensor([float("nan"), INF, -INF, 3e38], device="cuda")[torch.arange(n * K * V, device="cuda").reshape(n, K, V) % 4]
    logits = torch.where(mask.expand(n, K, V), logits, junk)
    check_select(logits, scores, finished=fin, mask=mask, eos=5, pad=1, keep_slots=True)
    check_select(logits, scores, finished=fin, mask=mask.to(torch.uint8) * 3, eos=5, pad=1)


@pytest.mark.parametrize("V", [51, 300, 2500])
def test_select_odd_values(V):
    """NaN, infinities and the types' lowest values where they are allowed; dead, finished and non-finite beams"""
    K = 8
    logits, scores, fin = make(6, K, V, seed=2, dead=0.0, done=0.0)
    logits[0, 1, 3], logits[0, 2, V - 1], logits[0, 4] = float("nan"), INF, -INF
    logits[1] = -INF                                                      # a group without continuations
    logits[2, 0], logits[2, 1, 1:] = torch.finfo(torch.float32).min, -INF  # every symbol at the lowest value; one symbol only
    logits[2, 2, ::2] = torch.finfo(torch.float32).min
    scores[3], fin[3, 5] = -INF, True                                     # finished but dead
    scores[4, 0], scores[4, 1], scores[4, 2] = float("nan"), INF, -INF
    fin[4, 0] = fin[5, :] = True
    logits[5] = float("nan")                                              # not looked at: all finished
    for keep in (False, True):
        check_select(logits, scores, finished=fin, eos=2, pad=0, keep_slots=keep)
    fin[3] = True
    got = check_select(logits, scores, finished=fin, keep_slots=True)
    assert got.finished[3].all() and torch.isinf(got.scores[3]).all()


@pytest.mark.parametrize("V", [7, 64, 513, 4100])
def test_select_ties_go_to_the_lowest_index(V):
    for dt in (torch.float32, torch.bfloat16):
        K = 8
        flat = torch.zeros(3, K, V, device="cuda", dtype=dt)
        scores = torch.zeros(3, K, device="cuda")
        got = check_select(flat, scores)
        assert got.parents[0].tolist() == [j // V for j in range(K)] and got.tokens[0].tolist() == [j % V for j in range(K)]
        check_select(flat, scores, keep_slots=True)
        # few distinct values: many ties inside a beam, and between beams of one score
        logits = torch.randint(0, 3, (5, K, V), generator=torch.Generator().manual_seed(V)).cuda().to(dt)
        logits[:, 1::2] = logits[:, ::2]
        check_select(logits, -torch.arange(5.0, device="cuda")[:, None].expand(5, K))
        fin = torch.zeros(5, K, device="cuda", dtype=torch.bool)
        fin[:, 1] = fin[:, 6] = True                                      # equal scores of finished beams
        check_select(logits, torch.full((5, K), -3.0, device="cuda"), finished=fin, pad=V - 1, keep_slots=True)
        check_select(flat, -0.0 * scores)


@pytest.mark.parametrize("V", [64, 128, 900, 3000, 20000])
def test_select_ties_made_by_rounding(V):
    """Logits that differ by less than the score's rounding: one score, so the lower index wins, not the larger logit"""
    K = 8
    up = 1.0 + torch.arange(V, device="cuda") * 2.0 ** -23        # the largest logits last
    logits = up.expand(6, K, V).contiguous()
    scores = torch.full((6, K), -1000.0, device="cuda")
    scores[1, 1:] = -INF                                           # one beam holds all winners
    scores[2, 3] = -900.0
    scores[3, 5], scores[3, 2] = -900.0, -901.0
    logits[4] = logits[4].flip(-1)
    logits[5, :, V // 3: V // 2] += 1e-4                           # part of them above the others' score
    for keep in (False, True):
        check_select(logits, scores, keep_slots=keep)
    got = check_select(logits[:1, :1].contiguous(), scores[:1, :1])   # K = 1: the argmax of the rounded scores
    assert got.tokens.item() == int(np.argmax(np.float32(-1000.0) + torch.log_softmax(up.double(), 0).float().cpu().numpy()))
    mask = torch.ones(V, device="cuda", dtype=torch.bool)
    mask[:5] = False
    check_select(logits, scores, mask=mask)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,K,V", [(9, 5, 51), (5, 8, 250), (4, 16, 900), (3, 8, 3000), (2, 7, 20000), (1, 16, 70000)])
def test_select_ties_between_and_within_beams(n, K, V, dt):
    """Scores so large that a step of their rounding spans many logits: most of what is compared is equal"""
    logits, scores, fin = make(n, K, V, dt, seed=7)
    for base in (-3.0e4, -1.0e6):
        s = torch.where(torch.isfinite(scores), scores.mul(0.05).round() + base, scores)
        check_select(logits, s, finished=fin, eos=1, keep_slots=True)
        check_select(logits, s[:, :1].expand(n, K))


def test_select_strides():
    logits, scores, fin = make(6, 5, 51, seed=3)
    wide = torch.full((6, 7, 80), float("nan"), device="cuda")
    wide[:, 1:6, 3:54] = logits
    check_select(wide[:, 1:6, 3:54], scores, finished=fin, eos=9)                               # rows of a wider buffer, odd start
    check_select(logits.permute(2, 0, 1).contiguous().permute(1, 2, 0), scores, finished=fin)   # vocabulary not dense: copied
    check_select(logits[:1].expand(6, 5, 51), scores, finished=fin, keep_slots=True)            # one group's logits for all
    check_select(logits, scores.t().contiguous().t(), finished=fin.t().contiguous().t())
    check_select(wide.bfloat16()[:, 1:6, 3:54], scores, finished=fin)
    m = torch.rand(12, 5, 102, device="cuda") < 0.5
    check_select(logits, scores, mask=m[::2, :, 1:52])
    assert vae.beam_select(logits[:0], scores[:0]).scores.shape == (0, 5)


def test_select_in_place_scores():
    """the C entry allows the new scores and flags over the old ones"""
    from polygon_amd.vae import beam
    for V in (51, 6000):
        logits, scores, fin = make(40, 8, V, seed=4)
        want = vae.beam_select(logits, scores, fin, eos=3, keep_slots=True)
        par, tok = torch.empty_like(want.parents), torch.empty_like(want.tokens)
        L = beam._entries()
        need = L.pg_beam_select_workspace_bytes(0, 40, 8, V)
        ws = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
        assert L.pg_beam_select(0, logits.data_ptr(), 8 * V, V, 40, 8, V, None, 0, 0, 1.0, scores.data_ptr(), fin.data_ptr(), 3, 0, 1,
                                scores.data_ptr(), par.data_ptr(), tok.data_ptr(), fin.data_ptr(), ws.data_ptr(), need,
                                torch.cuda.current_stream().cuda_stream) == 0
        for a, b in zip((scores, par, tok, fin), want):
            assert torch.equal(a, b)


# ---- pages ------------------------------------------------------------------------------------------------------------

def pool(P, widths=((512, torch.float32, 0), (512, torch.bfloat16, 0)), seed=0):
    """Planes [P, width] in rows `extra` elements wider, and the whole buffers behind them."""
    g = torch.Generator().manual_seed(seed)
    full = [(torch.randint(0, 255, (P, (w + e) * torch.empty(0, dtype=t).element_size()), generator=g).to(torch.uint8).cuda(), w, t)
            for w, t, e in widths]
    return [f.view(t)[:, :w] for f, w, t in full], [f for f, _, _ in full]


def raw(t):
    """a plane's pages as rows of bytes, on the host"""
    return t.contiguous().view(torch.uint8).reshape(t.shape[0], t[:1].numel() * t.element_size() if t.shape[0] else 1).cpu()


WIDTHS = [((512, torch.float32, 0), (512, torch.bfloat16, 0)), ((333, torch.bfloat16, 5), (7, torch.uint8, 0), (1, torch.uint8, 1)),
          ((3, torch.float32, 1), (2500, torch.float32, 0)), ((64, torch.float64, 2), (9000, torch.uint8, 7))]


@pytest.mark.parametrize("widths", WIDTHS)
@pytest.mark.parametrize("n,K", [(1, 1), (1, 5), (7, 8), (40, 9), (3, 32), (300, 4)])
def test_reorder(n, K, widths):
    planes, full = pool(n * K, widths)
    before = [f.cpu().clone() for f in full]
    old = [raw(p).clone() for p in planes]
    par = torch.randint(0, K, (n, K), generator=torch.Generator().manual_seed(n))
    par[0] = torch.arange(K).roll(1)                   # a cycle: every page is both source and target
    if n > 2:
        par[1], par[2] = K - 1, torch.arange(K)        # one source for all; nothing moves
    wild = par.clone()
    if n > 3:
        wild[3, 0], wild[3, -1] = -1, K                # out of range: stays
        par[3, 0], par[3, -1] = 0, K - 1
    vae.reorder_pages(planes, wild.int().cuda())
    rows = (par + torch.arange(n)[:, None] * K).flatten()
    for p, o, f, b, (w, t, e) in zip(planes, old, full, before, widths):
        assert torch.equal(raw(p), o[rows])
        used = w * t.itemsize
        assert torch.equal(f.cpu()[:, used:], b[:, used:])      # what lies between the rows is untouched


@pytest.mark.parametrize("widths", WIDTHS)
@pytest.mark.parametrize("P,Q", [(1, 1), (5, 1), (64, 8), (3, 200), (700, 700)])
def test_fork(P, Q, widths):
    dst, dfull = pool(P, widths, 1)
    src, sfull = pool(Q, widths, 2)
    index = torch.randint(0, Q, (P,), generator=torch.Generator().manual_seed(P))
    wild = index.clone()
    if P > 4:
        wild[1], wild[3] = -5, Q
    before, kept = [raw(d).clone() for d in dst], [f.cpu().clone() for f in dfull]
    unread = [f.cpu().clone() for f in sfull]
    vae.fork_pages(dst, src, wild.int().cuda())
    stays = (wild < 0) | (wild >= Q)
    for d, s, b, f, k, (w, t, e) in zip(dst, src, before, dfull, kept, widths):
        want = torch.where(stays[:, None], b, raw(s)[index])
        assert torch.equal(raw(d), want)
        assert torch.equal(f.cpu()[:, w * t.itemsize:], k[:, w * t.itemsize:])
    assert all(torch.equal(f.cpu(), u) for f, u in zip(sfull, unread))


def ref_compact(live):
    live = live.cpu().numpy()
    count = int(live.sum())
    where = np.where(live, np.arange(live.size), -1).astype(np.int32)
    where[np.flatnonzero(live[count:]) + count] = np.flatnonzero(~live[:count])
    return count, where


@pytest.mark.parametrize("share", [0.0, 0.03, 0.5, 0.97, 1.0])
@pytest.mark.parametrize("P,widths", [(0, WIDTHS[0]), (1, WIDTHS[0]), (8, WIDTHS[1]), (63, WIDTHS[2]), (1025, WIDTHS[1]), (4096, WIDTHS[1]),
                                      (5000, WIDTHS[0]), (16385, ((3, torch.uint8, 0),)), (70001, ((5, torch.float32, 0),)),
                                      (300000, ((1, torch.float32, 0),))])
def test_compact(P, widths, share):
    planes, full = pool(P, widths)
    live = (torch.rand(P, generator=torch.Generator().manual_seed(P)) < share).cuda()
    old, kept = [raw(p).clone() for p in planes], [f.cpu().clone() for f in full]
    count, where = vae.compact_pages(planes, live)
    c, w = ref_compact(live)
    assert count.tolist() == [c] and np.array_equal(where.cpu().numpy(), w)
    src = np.flatnonzero(w >= 0)
    for p, o, f, k, (wd, t, e) in zip(planes, old, full, kept, widths):
        want = o.clone()
        want[torch.from_numpy(w[src]).long()] = o[torch.from_numpy(src)]
        assert torch.equal(raw(p), want)
        assert torch.equal(f.cpu()[:, wd * t.itemsize:], k[:, wd * t.itemsize:])


def test_compact_one_edge():
    for live in ([0, 0, 0, 1], [1, 0, 0, 0], [0, 1, 0, 1], [1, 1, 1, 0], [0, 1, 1, 1]):
        planes, _ = pool(4, ((2, torch.uint8, 0),))
        old = planes[0].cpu().clone()
        t = torch.tensor(live, dtype=torch.uint8, device="cuda") * 200
        count, where = vae.compact_pages(planes, t)
        c, w = ref_compact(t != 0)
        assert count.item() == c and where.tolist() == w.tolist()
        for p, q in enumerate(w):
            if q >= 0:
                assert torch.equal(planes[0][q].cpu(), old[p])


def test_interleaved_planes():
    """two planes in one buffer, a page of the second right behind the first's"""
    both = torch.randn(12, 2, 100, device="cuda")
    old = both.clone()
    par = torch.tensor([[1, 0, 1], [2, 2, 2], [0, 1, 2], [2, 1, 0]], dtype=torch.int32, device="cuda")
    vae.reorder_pages([both[:, 0], both[:, 1]], par)
    assert torch.equal(both, old[(par.cpu() + torch.arange(4)[:, None] * 3).flatten()])
    with pytest.raises(PolygonHipError):
        vae.reorder_pages([both[:, 0], both[:, 0]], par)
    with pytest.raises(PolygonHipError):
        vae.fork_pages([both[:6, 0]], [both[5:, 0]], torch.zeros(6, dtype=torch.int32, device="cuda"))
    vae.fork_pages([both[:, 0]], [both[:, 1]], torch.arange(12, dtype=torch.int32, device="cuda"))
    assert torch.equal(both[:, 0], both[:, 1])


def test_indices_between_and_inside_pages():
    """flags and parents that share a buffer with the pages: taken where they lie beside them, refused where they are moved too"""
    full = torch.randint(0, 200, (12, 128), device="cuda", dtype=torch.uint8)
    old = full.cpu().clone()
    live, par = full[2, 64:76], full[5, 68:116].view(torch.int32).view(3, 4)
    flags = torch.tensor([1, 0, 0, 1, 1, 0, 1, 0, 1, 1, 0, 1], dtype=torch.uint8)
    live.copy_(flags)
    old[2, 64:76] = flags
    c, w = ref_compact(flags != 0)
    count, where = vae.compact_pages([full[:, :64]], live)
    for p, q in enumerate(w):
        if q >= 0:
            old[q, :64] = old[p, :64]
    assert count.item() == c and where.tolist() == w.tolist() and torch.equal(full[:c, :64].cpu(), old[:c, :64])
    par.copy_(torch.tensor([[1, 1, 2, 0], [0, 1, 2, 3], [3, 2, 1, 0]], dtype=torch.int32))
    old, rows = full.cpu().clone(), (par.cpu() + torch.arange(3)[:, None] * 4).flatten()
    vae.reorder_pages([full[:, :64]], par)
    assert torch.equal(full[:, :64].cpu(), old[rows][:, :64]) and torch.equal(full[:, 64:].cpu(), old[:, 64:])

    state, alive = torch.randn(6, 40, device="cuda"), torch.ones(6, dtype=torch.bool, device="cuda")
    parents, other = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    index = torch.zeros(6, dtype=torch.int32, device="cuda")
    with pytest.raises(PolygonHipError):
        vae.compact_pages([state, alive], alive)
    with pytest.raises(PolygonHipError):
        vae.reorder_pages([state, parents.view(6)], parents)
    with pytest.raises(PolygonHipError):
        vae.fork_pages([index], [other], index)
    vae.compact_pages([state, alive], alive.clone())
    vae.fork_pages([other], [index], index)               # only read: may be a page


def test_far_offsets():
    """pages beyond 2^31 and 2^32 bytes"""
    P = 70000
    plane = torch.zeros(P, 65536, device="cuda", dtype=torch.uint8)
    plane[P - 8:] = torch.arange(8, device="cuda", dtype=torch.uint8)[:, None] + 1
    par = torch.arange(8, device="cuda", dtype=torch.int32).repeat(P // 8, 1)
    par[-1] = torch.tensor([7, 1, 2, 3, 4, 5, 6, 0])
    vae.reorder_pages([plane], par)
    assert plane[P - 8:, ::997].float().mean(1).tolist() == [8, 2, 3, 4, 5, 6, 7, 1]
    out = torch.zeros(2, 65536, device="cuda", dtype=torch.uint8)
    vae.fork_pages([out], [plane], torch.tensor([P - 1, P - 3], dtype=torch.int32, device="cuda"))
    assert (out[0] == 1).all() and (out[1] == 6).all()
    live = torch.zeros(P, device="cuda", dtype=torch.bool)
    live[P - 2:] = True
    count, where = vae.compact_pages([plane], live)
    assert count.item() == 2 and where[P - 2:].tolist() == [0, 1] and (plane[0] == 7).all() and (plane[1] == 1).all()


def test_select_far_offsets():
    """logits whose last group starts beyond 2^32 bytes"""
    n, K, V = 66, 32, 1 << 19
    logits = torch.zeros(n, K, V, device="cuda")
    logits[-1, 30, 12345] = 9.0
    logits[-1, 31, V - 1] = 8.0
    scores = torch.zeros(n, K, device="cuda")
    got = vae.beam_select(logits[-1:], scores[:1])
    all_ = vae.beam_select(logits, scores)
    assert all_.tokens[-1, :2].tolist() == [12345, V - 1] and all_.parents[-1, :2].tolist() == [30, 31]
    assert all(torch.equal(a[0], b[-1]) for a, b in zip(got, all_))


# ---- as they are used ---------------------------------------------------------------------------------------------------

def test_stream_and_graph():
    """one step (selection, reorder, compaction) on another stream, and captured: replays with new inputs match eager calls"""
    n, K, V = 37, 6, 51

    def step(logits, scores, fin, planes, live):
        s = vae.beam_select(logits, scores, fin, eos=2, keep_slots=True)
        vae.reorder_pages(planes, s.parents)
        return list(s) + list(vae.compact_pages([p.view(n, -1) for p in planes], live))

    def inputs(seed):
        logits, scores, fin = make(n, K, V, seed=seed)
        return [logits, scores, fin, pool(n * K, WIDTHS[0], seed)[0], torch.rand(n, generator=torch.Generator().manual_seed(seed)).cuda() < 0.6]

    wide = torch.randn(2, 4, 20000, device="cuda")
    a = inputs(0)
    a[3] = [p.clone() for p in a[3]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(*a)
        w0 = vae.beam_select(wide, torch.zeros(2, 4, device="cuda"))
    torch.cuda.current_stream().wait_stream(side)
    static = inputs(0)
    static[3] = [p.clone() for p in static[3]]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = step(*static)
        w1 = vae.beam_select(wide, torch.zeros(2, 4, device="cuda"))
    for seed in (0, 5, 6, 7):
        fresh = inputs(seed)
        for d, s in zip(static[:3] + static[3] + static[4:], fresh[:3] + fresh[3] + fresh[4:]):
            d.copy_(s)
        wide.add_(0.25 * seed)
        graph.replay()
        want = step(*fresh)
        w2 = vae.beam_select(wide, torch.zeros(2, 4, device="cuda"))
        torch.cuda.synchronize()
        for x, y in zip(outs + static[3] + list(w1), want + fresh[3] + list(w2)):
            assert torch.equal(x.view(torch.uint8) if x.dtype.is_floating_point else x, y.view(torch.uint8) if y.dtype.is_floating_point else y)
        if seed == 0:
            assert all(torch.equal(x, y) for x, y in zip(first, want)) and all(torch.equal(x, y) for x, y in zip(w0, w2))


def test_same_call_same_bits():
    for V in (51, 9000):
        logits, scores, fin = make(50, 8, V, seed=9)
        a = vae.beam_select(logits, scores, fin, keep_slots=True)
        for _ in range(3):
            assert all(torch.equal(x, y) for x, y in zip(a, vae.beam_select(logits, scores, fin, keep_slots=True)))
