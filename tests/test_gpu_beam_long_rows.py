"""Selection over long vocabularies with enough rows that a wave walks through several tiles of 1024 symbols: the running sum is
rescaled from tile to tile, the bound of the best so far is the last ranking's, later tiles append behind a ranked list.  Compared
with the 64-bit definition for some groups of every call (the first and the last among them)."""
import numpy as np
import pytest
import torch

from polygon_amd import vae
from tests.test_gpu_beam_ops import INF, make, ref_select

pytestmark = pytest.mark.gpu

# n, K, V: rows * tiles of 1024 symbols of at least 8192 give a chunk more than one tile
SHAPES = [(300, 8, 5003), (64, 32, 9000), (32, 32, 33333), (4100, 1, 20011), (600, 16, 3000)]


def check_some(logits, scores, finished=None, mask=None, **kw):
    n = logits.shape[0]
    got = vae.beam_select(logits, scores, finished=finished, mask=mask, **kw)
    pick = torch.tensor(sorted({0, 1, n // 2, n - 1}))
    sub = lambda t: None if t is None else t[pick.to(t.device)]  # noqa: E731
    want = ref_select(sub(logits), sub(scores), sub(finished), mask if mask is None or mask.dim() == 1 else sub(mask), **kw)
    for name, a, b in zip(got._fields[1:], got[1:], want[1:]):
        assert np.array_equal(sub(a).cpu().numpy(), b), name
    a, b, s = sub(got.scores).cpu().numpy(), want[0], sub(scores).cpu().numpy()
    f = np.isfinite(b)
    assert np.array_equal(np.isfinite(a), f)
    # the log-probability and its sum with the score are rounded once each; two 64-bit values next to a rounding's edge may go to
    # either side: one step (2^-23 of the value) of each
    lim = 2.0 ** -23 * (2 * np.abs(b[f]) + np.abs(s[np.isfinite(s)]).max(initial=0.0))
    assert (np.abs(a[f] - b[f]) <= lim).all()
    return got


def arrange(kind, logits, seed):
    """random logits in an order along the vocabulary that a walk through tiles meets differently"""
    n, K, V = logits.shape
    if kind == "ascending":                # every tile beats all before it
        return logits.sort(-1).values
    if kind == "descending":               # the first tile holds everything
        return logits.sort(-1, descending=True).values
    if kind == "few":                      # three values: ties all over, over tiles
        return logits.sign().mul((logits.abs() > 1.0).to(logits.dtype))
    if kind == "late":                     # nothing before the last tiles, and a maximum that moves up in jumps
        x = logits - 60.0
        x[..., V // 2:] += 25.0
        x[..., V - V // 8:] += 40.0
        x[::2, :, : V // 3] = -INF
        return x
    if kind == "rare":                     # each tile a handful above the best so far
        g = torch.Generator().manual_seed(seed)
        x = torch.full_like(logits, -8.0)
        x[..., torch.randperm(V, generator=g)[: max(64, V // 50)].cuda()] = 0
        return x + logits * (x == 0) + torch.arange(V, device="cuda") / V
    return logits


@pytest.mark.parametrize("kind", ["random", "ascending", "descending", "few", "late", "rare"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,K,V", SHAPES)
def test_tiles_of_a_chunk(n, K, V, dt, kind):
    logits, scores, fin = make(n, K, V, dt, seed=11, dead=0.05)
    x = arrange(kind, logits, V).to(dt).contiguous()
    check_some(x, scores, finished=fin, eos=V - 1, pad=V // 2, keep_slots=True)
    check_some(x, scores, temp=0.6)


@pytest.mark.parametrize("n,K,V", SHAPES)
def test_masks_over_tiles(n, K, V):
    logits, scores, fin = make(n, K, V, torch.bfloat16, seed=12)
    g = torch.Generator().manual_seed(V)
    row = (torch.rand(K, V, generator=g) < 0.5).cuda().expand(n, K, V)
    junk = torch.where(row, logits, torch.full_like(logits, float("nan")))
    check_some(junk, scores, finished=fin, mask=row, eos=3, keep_slots=True)
    last = torch.zeros(V, dtype=torch.bool, device="cuda")
    last[-5:] = True                                        # only the last tile has anything
    check_some(logits, scores, mask=last, keep_slots=True)
    rows = torch.ones(n, K, 1, dtype=torch.bool, device="cuda")
    rows[0, 0] = rows[-1, -1] = False                       # rows that nothing is left of
    check_some(logits, scores, mask=rows & (torch.arange(V, device="cuda") % 7 != 2), pad=2)


@pytest.mark.parametrize("n,K,V", SHAPES)
def test_odd_values_in_later_tiles(n, K, V):
    """a NaN or +inf that only a later tile of a row holds takes the row's continuations away; -inf and the lowest number do not"""
    logits, scores, fin = make(n, K, V, seed=13, dead=0.0, done=0.0)
    low = torch.finfo(torch.float32).min
    logits[0, 0, V - 3], logits[1, 0, 2000] = float("nan"), INF
    logits[n // 2, -1, 1500], logits[-1, 0, V - 1] = -INF, low
    logits[-1, -1, :2500] = low
    logits[n - 1, K // 2, 1100:] = -INF
    for keep in (False, True):
        got = check_some(logits, scores, eos=1, keep_slots=keep)
    if K == 1:
        assert torch.isinf(got.scores[:2]).all() and torch.isfinite(got.scores[2:]).all()


@pytest.mark.parametrize("base", [-1.0e3, -1.0e6])
@pytest.mark.parametrize("n,K,V", SHAPES)
def test_rounding_ties_over_tiles(n, K, V, base):
    """logits closer than a score's rounding, the largest last: the lower index wins although its logit is the smaller one"""
    near = 1.0 + torch.arange(V, device="cuda") * 2.0 ** -23
    logits = near.expand(n, K, V).clone()
    logits[1::2] = logits[1::2].flip(-1)
    scores = torch.full((n, K), base, device="cuda")
    scores[0, K // 2:] -= 1.0
    check_some(logits, scores, keep_slots=True)
    logits[:, :, V // 3: V // 3 + 3] += 1e-3                # three clear winners a beam, the rest tied
    check_some(logits, scores)


def test_scores_in_place_and_same_bits():
    from polygon_amd.vae import beam
    n, K, V = 300, 8, 5003
    logits, scores, fin = make(n, K, V, seed=14)
    want = vae.beam_select(logits, scores, fin, eos=3, keep_slots=True)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(want, vae.beam_select(logits, scores, fin, eos=3, keep_slots=True)))
    L = beam._entries()
    need = L.pg_beam_select_workspace_bytes(0, n, K, V)
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    par, tok = torch.empty_like(want.parents), torch.empty_like(want.tokens)
    assert L.pg_beam_select(0, logits.data_ptr(), K * V, V, n, K, V, None, 0, 0, 1.0, scores.data_ptr(), fin.data_ptr(), 3, 0, 1,
                            scores.data_ptr(), par.data_ptr(), tok.data_ptr(), fin.data_ptr(), ws.data_ptr(), need,
                            torch.cuda.current_stream().cuda_stream) == 0
    assert all(torch.equal(a, b) for a, b in zip((scores, par, tok, fin), want))
