"""VAE.beam_search against the per-step sampler's own probabilities, which it computes for given strings (teacher forcing) with the
same cells: bf16 as closely as fp32, and vocabularies of 65 to 128 symbols at every step.

Tolerance of a step's log-probability.  u = 2^-24, A = the largest sum of |weights| and |bias| of a symbol (|h| < 1), H units, V symbols.
Both sides accumulate a logit's H products in fp32, in other orders: 2 (H + 2) u A between them, twice that in a log-softmax.  The
sampler's softmax in fp32: the exponent's difference (at most 2 A) is rounded and scaled, three roundings, the exponential is off by
2^-22 = 4 u, for the symbol and for the sum alike; V additions and a division.  A score rounds the log-probability and the sum."""
import numpy as np
import pytest
import torch

from polygon_amd import _lib
from polygon_amd.utils.moses_utils import OneHotVocab
from polygon_amd.vae.vae_model import VAE
from tests.helpers import REAL, TINY

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def per_step_sampler():
    old = _lib.lib().pg_persist_disable(-1)
    _lib.lib().pg_persist_disable(15)
    yield
    _lib.lib().pg_persist_disable(old)


def make_model(dims, symbols, dt, mul, eos, seed=5):
    torch.manual_seed(seed)
    vocab = dict(vocabulary=OneHotVocab([chr(200 + i) for i in range(symbols - 4)])) if symbols else {}
    model = VAE(q_d_h=dims["Hq"], d_z=dims["Dz"], d_d_h=dims["Hd"], d_n_layers=dims["L"], compute_dtype=dt, **vocab).cuda()
    with torch.no_grad():
        model.decoder_fc.weight.mul_(mul)
        model.decoder_fc.bias[model.eos] += eos
    return model


def step_tolerance(model):
    w, b = model.decoder_fc.weight.detach().double().cpu(), model.decoder_fc.bias.detach().double().cpu()
    V, H = w.shape
    A = float((w.abs().sum(1) * (1 + 2.0 ** -8) + b.abs()).max())            # (1 + 2^-8: weights rounded to bf16)
    return lambda s, lp: U * (4 * (H + 2) * A + 2 * (3 * 2 * A + 4) + V + 3 + np.abs(lp) + np.abs(s))


def log_probs(model, z, tokens):
    """[steps, rows, V]: of every symbol at every step, behind the tokens before it"""
    n, T = tokens.shape
    p = model.sample_tokens(n, max_len=T, z=z, forced=tokens, return_probs=True, seed=0)[2]
    return p[:, :, :len(model.vocabulary)].double().log().cpu().numpy()


CASES = [(TINY, 0, 3, 40, 26), (TINY, 0, 8, 40, 34), (TINY, 0, 20, 16, 20), (TINY, 96, 4, 30, 22), (TINY, 128, 8, 30, 30), (TINY, 65, 12, 20, 18),
         (TINY, 96, 32, 9, 18), (REAL, 0, 8, 6, 18), (REAL, 96, 32, 3, 12)]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("eos", [0.0, 1.0])
@pytest.mark.parametrize("dims,symbols,K,n,T", CASES)
def test_scores_are_the_samplers_probabilities(dims, symbols, K, n, T, eos, dt):
    """eos 0: most strings reach the end; 1: most end before, and their latents leave"""
    model = make_model(dims, symbols, dt, 2.0, eos)
    z = torch.randn(n, dims["Dz"], generator=torch.Generator().manual_seed(n)).cuda()
    tok, end, sc = model.beam_search_tokens(z, K, T)
    lp = log_probs(model, z.repeat_interleave(K, 0), tok.view(n * K, T))
    tok, end, sc = tok.view(n * K, T).cpu().numpy().astype(int), end.view(-1).cpu().numpy(), sc.view(-1).double().cpu().numpy()
    tol, want, room, rows = step_tolerance(model), np.zeros(n * K), np.zeros(n * K), np.arange(n * K)
    assert np.isfinite(sc).all()
    for i in range(1, T):
        inside = i < end
        step = np.where(inside, lp[i - 1, rows, tok[:, i]], 0.0)
        want += step
        room += np.where(inside, tol(want, step), 0.0)
    assert (np.abs(sc - want) <= room).all(), float(np.abs(sc - want).max())


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("dims,symbols,K,n,T", [(TINY, 0, 3, 120, 18), (TINY, 0, 8, 120, 9), (TINY, 96, 4, 120, 12), (TINY, 128, 6, 300, 6),
                                                (TINY, 70, 9, 200, 5), (REAL, 96, 3, 120, 5)])
def test_search_over_the_samplers_probabilities(dims, symbols, K, n, T, dt):
    """a plain search in 64 bits that asks the sampler for every step's probabilities finds the same strings, where every step of
    it was decided by more than the two can differ"""
    model = make_model(dims, symbols, dt, 10.0, 1.0)
    V = len(model.vocabulary)
    z = torch.randn(n, dims["Dz"], generator=torch.Generator().manual_seed(n + 1)).cuda()
    tol, zr = step_tolerance(model), z.repeat_interleave(K, 0)
    strings = np.full((n, K, T), model.pad)
    strings[:, :, 0] = model.bos
    s, room = np.full((n, K), -np.inf), np.zeros((n, K))
    s[:, 0] = 0.0
    fin, sure = np.zeros((n, K), bool), np.ones(n, bool)
    for i in range(1, T):
        fed = torch.from_numpy(strings.reshape(n * K, T).astype(np.uint8)).cuda()
        lp = log_probs(model, zr, fed)[i - 1].reshape(n, K, V)
        for g in range(n):
            cand = []
            for k in np.flatnonzero(np.isfinite(s[g])):
                if fin[g, k]:
                    cand.append((s[g, k], k, model.pad, room[g, k]))
                else:
                    cand += [(s[g, k] + lp[g, k, v], k, v, room[g, k] + tol(s[g, k] + lp[g, k, v], lp[g, k, v]))
                             for v in np.argsort(-lp[g, k])[:K + 1]]
            cand.sort(key=lambda c: -c[0])
            sure[g] &= all(a[0] - b[0] > a[3] + b[3] for a, b in zip(cand[:K], cand[1:K + 1]))
            old = strings[g].copy(), fin[g].copy()
            s[g] = -np.inf
            for j, (c, k, v, r) in enumerate(cand[:K]):
                strings[g, j], s[g, j], room[g, j] = old[0][k], c, r
                strings[g, j, i] = v
                fin[g, j] = old[1][k] or v == model.eos
    tok, end, sc = [t.cpu().numpy() for t in model.beam_search_tokens(z, K, T)]
    assert sure.sum() >= 3 and end[sure].max() >= 4, "too few of the searches are clearly decided"
    assert np.array_equal(tok[sure], strings[sure]) and (np.abs(sc[sure] - s[sure]) <= room[sure]).all()


SHAPES = [(dict(Hq=32, Dz=8, Hd=32, L=1), 0), (dict(Hq=32, Dz=24, Hd=96, L=2), 0), (dict(Hq=64, Dz=40, Hd=160, L=8), 0),
          (dict(Hq=32, Dz=8, Hd=32, L=2), 100), (dict(Hq=32, Dz=16, Hd=224, L=4), 66), (dict(Hq=32, Dz=16, Hd=64, L=1), 5)]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("dims,symbols", SHAPES)
def test_decoder_shapes(dims, symbols, dt):
    """hidden sizes that no tile divides, one layer to eight, a vocabulary of five; one beam and as many as there are"""
    model = make_model(dims, symbols, dt, 2.0, 0.5)
    for K, n, T in ((1, 70, 20), (7, 33, 19), (32, 5, 10)):
        z = torch.randn(n, dims["Dz"], generator=torch.Generator().manual_seed(K)).cuda()
        tok, end, sc = model.beam_search_tokens(z, K, T)
        lp = log_probs(model, z.repeat_interleave(K, 0), tok.view(n * K, T))
        tok, end, sc = tok.view(n * K, T).cpu().numpy().astype(int), end.view(-1).cpu().numpy(), sc.view(-1).double().cpu().numpy()
        tol, want, room, rows = step_tolerance(model), np.zeros(n * K), np.zeros(n * K), np.arange(n * K)
        assert np.isfinite(sc).all() or symbols == 5
        for i in range(1, T):
            inside = i < end
            step = np.where(inside, lp[i - 1, rows, tok[:, i]], 0.0)
            want += step
            room += np.where(inside, tol(want, step), 0.0)
        has = np.isfinite(sc)
        assert (np.abs(sc - want)[has] <= room[has]).all(), (K, float(np.abs(sc - want)[has].max()))
        assert (end[~has] == 0).all()
        assert all(len({tuple(t) for t, e in zip(tok[g * K:g * K + K], end[g * K:]) if e}) == has[g * K:g * K + K].sum() for g in range(n))
