"""VAE.beam_search against a plain float64 beam search over the CPU oracle's decoder, and its properties at the sizes and
masks where it could go wrong.

Tolerances: the logits of a given string are held to TOL * max |y| (the parity bound: 1e-3 for fp32, 2e-2 for bf16).  A
log-softmax moves by at most the shift of its own logit plus the largest shift of any (its normaliser is an average), so a
score, their sum over a string's symbols, is off by at most the sum of 2 TOL max |y| over its steps.  Strings are compared where the oracle's own search is decided by more than those errors can move: 1e-3 nats
between what a step keeps and what it drops (fp32; its errors are some 1e-6)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import vae_oracle as O
from polygon_amd import _lib
from tests.helpers import REAL, TINY, build_model

pytestmark = pytest.mark.gpu
TOL = {"fp32": 1e-3, "bf16": 2e-2}


def sharp_model(dims, seed, dt, mul=20.0, eos=2.0):
    """A head `mul` times the initial one: distributions with clear favourites, about half of the latents' beams ending after 3 to
    20 symbols and the others running on."""
    model, P = build_model(dims, seed, dt, eos_bias=eos)
    with torch.no_grad():
        model.decoder_fc.weight.mul_(mul)
    P["decoder_fc.weight"] = P["decoder_fc.weight"] * mul
    return model, P


class OracleDecoder:
    """The oracle's decoder one step at a time, rows picked by the caller."""

    def __init__(self, P, z):
        self.P, self.L = P, O.n_decoder_layers(P)
        self.z = z
        self.h = [z @ P["decoder_lat.weight"].T + P["decoder_lat.bias"] for _ in range(self.L)]

    def pick(self, rows):
        self.z, self.h = self.z[rows], [h[rows] for h in self.h]

    def step(self, w, temp=1.0):
        P = self.P
        inp = np.concatenate([P["x_emb.weight"][w], self.z], axis=1)
        for l in range(self.L):
            gi = inp @ P["decoder_rnn.weight_ih_l%d" % l].T + P["decoder_rnn.bias_ih_l%d" % l]
            gh = self.h[l] @ P["decoder_rnn.weight_hh_l%d" % l].T + P["decoder_rnn.bias_hh_l%d" % l]
            self.h[l], _ = O.gru_cell(gi, gh, self.h[l])
            inp = self.h[l]
        return (inp @ P["decoder_fc.weight"].T + P["decoder_fc.bias"]) / temp


def log_softmax(y):
    y = y - y.max(1, keepdims=True)
    return y - np.log(np.exp(y).sum(1, keepdims=True))


def oracle_scores(P, z, tokens, ends, temp=1.0, allowed=None):
    """Sum of log-probabilities of given rows [n, T] (z [n, Dz]) up to their end positions, and of the steps' max |logit|."""
    dec, out, size = OracleDecoder(P, z), np.zeros(len(z)), np.zeros(len(z))
    for i in range(1, tokens.shape[1]):
        y = dec.step(tokens[:, i - 1], temp)
        size += np.where(i < ends, np.abs(y).max(1), 0.0)
        if allowed is not None:
            y = np.where(allowed, y, -np.inf)
        out += np.where(i < ends, log_softmax(y)[np.arange(len(z)), tokens[:, i]], 0.0)
    return out, size


def oracle_beam(P, z, K, max_len, temp=1.0):
    """One latent: [(score, tokens)] best first, and the narrowest margin by which a step decided."""
    dec = OracleDecoder(P, z[None])
    beams, margin = [(0.0, [O.BOS], False)], np.inf
    for _ in range(1, max_len):
        lp = log_softmax(dec.step(np.array([b[1][-1] for b in beams]), temp))
        cand = []
        for k, (s, t, fin) in enumerate(beams):
            if fin:
                cand.append((s, k, None))
            else:
                cand += [(s + lp[k, v], k, v) for v in range(lp.shape[1])]
        cand.sort(key=lambda c: -c[0])
        s = [c[0] for c in cand[:K + 1]]
        margin = min([margin] + [a - b for a, b in zip(s, s[1:])])
        dec.pick([c[1] for c in cand[:K]])
        beams = [(s, beams[k][1] + [O.PAD if v is None else v], beams[k][2] or v == O.EOS) for s, k, v in cand[:K]]
        if all(b[2] for b in beams):
            break
    return beams, margin


def check_scores(P, z, out, dt, temp=1.0, allowed=None):
    tok, end, sc = [t.cpu().numpy() for t in out]
    n, K, T = tok.shape
    has = np.isfinite(sc).reshape(-1)
    want, size = oracle_scores(P, np.repeat(z.astype(np.float64), K, 0)[has], tok.reshape(n * K, T)[has].astype(np.int64),
                               end.reshape(-1)[has], temp, allowed)
    assert bool((np.abs(sc.reshape(-1)[has] - want) <= 2 * TOL[dt] * size).all())
    assert (np.diff(np.where(np.isfinite(sc), sc, -1e30), axis=1) <= 0).all()           # best first
    assert (tok[:, :, 0] == O.BOS).all()
    for i in range(n):
        rows = [tuple(tok[i, j, :end[i, j]]) for j in range(K) if np.isfinite(sc[i, j])]
        assert len(set(rows)) == len(rows)                                              # different hypotheses
        for j in range(K):
            e = end[i, j]
            assert (e == 0) == (not np.isfinite(sc[i, j])) and (tok[i, j, max(e, 1):] == O.PAD).all()
            assert e in (0, T) or tok[i, j, e - 1] == O.EOS
            assert O.EOS not in tok[i, j, 1:max(e - 1, 1)]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("dims,n,K,max_len,eos", [(TINY, 5, 4, 12, 0.0), (TINY, 40, 8, 30, 3.0), (TINY, 3, 32, 20, 2.0), (TINY, 7, 1, 25, 2.0),
                                                  (TINY, 600, 13, 40, 3.5), (REAL, 6, 5, 24, 3.0), (REAL, 2, 16, 9, 0.0)])
def test_scores_are_the_strings_log_probabilities(dims, n, K, max_len, eos, dt):
    model, P = build_model(dims, 21, dt, eos_bias=eos)
    z = np.random.default_rng(n).standard_normal((n, dims["Dz"])).astype(np.float32)
    check_scores(P, z, model.beam_search_tokens(torch.from_numpy(z), K, max_len), dt)
    if K in (5, 13):
        check_scores(P, z, model.beam_search_tokens(torch.from_numpy(z), K, max_len, temp=0.8), dt, temp=0.8)


@pytest.mark.parametrize("dims,n,K,max_len,eos", [(TINY, 24, 4, 14, 2.0), (TINY, 12, 9, 20, 3.0), (REAL, 8, 5, 16, 2.5)])
def test_matches_the_oracles_search(dims, n, K, max_len, eos):
    model, P = sharp_model(dims, 33, "fp32", 12.0, eos)
    z = np.random.default_rng(5).standard_normal((n, dims["Dz"])).astype(np.float32)
    tok, end, sc = [t.cpu().numpy() for t in model.beam_search_tokens(torch.from_numpy(z), K, max_len)]
    strings, scores = model.beam_search(torch.from_numpy(z), K, max_len)
    sure = 0
    for i in range(n):
        beams, margin = oracle_beam(P, z[i].astype(np.float64), K, max_len)
        if margin < 1e-3:
            continue
        sure += 1
        for j, (s, t, fin) in enumerate(beams):
            e = t.index(O.EOS) + 1 if fin else max_len
            assert end[i, j] == e and tok[i, j, :e].tolist() == t[:e]
            assert abs(sc[i, j] - s) <= 1e-3         # (the margin above: a larger error could have changed the strings)
            assert strings[i][j] == O.ids2string(t[:e])
    assert sure >= 3, "too few of the oracle's searches are clearly decided"
    assert torch.equal(scores, torch.from_numpy(sc))


def test_one_beam_is_greedy():
    model, P = build_model(TINY, 8, "fp32", eos_bias=2.0)
    z = torch.randn(33, TINY["Dz"], generator=torch.Generator().manual_seed(1))
    assert [s[0] for s in model.beam_search(z, 1, max_len=20)[0]] == model.sample(33, max_len=20, z=z, multinomial=False)
    assert model.decode(z, beam_width=1) == model.sample(33, z=z, multinomial=False)
    wide, sc = model.beam_search(z, 8, max_len=20)
    one = model.beam_search(z, 1, max_len=20)[1]
    assert (sc[:, 0] >= one[:, 0] - 1e-4).float().mean() > 0.9      # (not always: a search may drop the greedy prefix)
    assert len(wide) == 33 and all(len(s) == 8 for s in wide)
    assert model.decode(z, beam_width=8) == [s[0] for s in model.beam_search(z, 8)[0]]
    with pytest.raises(ValueError):
        model.decode(z, x=[model.string2tensor("CC")] * 33, beam_width=2)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_allowed_symbols(dt):
    model, P = build_model(TINY, 4, dt, eos_bias=1.0)
    V = len(model.vocabulary)
    z = torch.randn(9, TINY["Dz"], generator=torch.Generator().manual_seed(2))
    ok = torch.ones(V, dtype=torch.bool)
    ok[[model.pad, model.bos, model.unk]] = False
    out = model.beam_search_tokens(z, 6, 15, allowed=ok)
    tok, end = out[0].cpu(), out[1].cpu()
    for i in range(9):
        for j in range(6):
            assert ok[tok[i, j, 1:end[i, j]].long()].all()
    check_scores(P, z.numpy(), out, dt, allowed=ok.numpy())
    # two symbols and two positions: bos x, x in {C, eos}, then the second symbol: 3 strings of at most 2 symbols end or reach max_len
    c = model.vocabulary.c2i["C"]
    ok = torch.zeros(V, dtype=torch.uint8)
    ok[[c, model.eos]] = 1
    strings, sc = model.beam_search(z, 8, max_len=3, allowed=ok)
    for i in range(9):
        assert sorted(strings[i]) == [""] * 6 + ["C", "CC"] and torch.isfinite(sc[i]).sum() == 3
        # eos; C eos; C C: the probabilities of all there is
        assert abs(sc[i].double().exp().sum().item() - 1.0) <= (1e-4 if dt == "fp32" else 1e-4)
    ok[c] = 0
    strings, sc = model.beam_search(z, 3, max_len=40, allowed=ok)
    assert strings == [[""] * 3] * 9 and torch.equal(sc[:, 0], torch.zeros(9)) and torch.isinf(sc[:, 1:]).all()
    ok[model.eos] = 0
    strings, sc = model.beam_search(z, 3, max_len=7, allowed=ok)          # nothing may be taken
    assert strings == [[""] * 3] * 9 and torch.isinf(sc).all()


def test_wide_vocabulary_and_shortest():
    from polygon_amd.utils.moses_utils import OneHotVocab
    from polygon_amd.vae.vae_model import VAE
    torch.manual_seed(3)
    model = VAE(vocabulary=OneHotVocab([chr(200 + i) for i in range(90)]), q_d_h=32, d_z=16, d_d_h=64, d_n_layers=2).cuda()
    z = torch.randn(11, 16)
    for K in (3, 8, 20):
        tok, end, sc = model.beam_search_tokens(z, K, 10)
        assert torch.isfinite(sc).all() and (tok[:, :, 0] == model.bos).all()
        two = model.beam_search_tokens(z, K, 2)
        assert two[0].shape == (11, K, 2) and (two[2] <= 0).all() and (two[2].diff(dim=1) <= 0).all()
    # one step: the K most probable first symbols
    p = model.sample_tokens(11, max_len=2, z=z, return_probs=True, seed=0)[2][0][:, :len(model.vocabulary)]
    assert torch.equal(two[0][:, :, 1].long(), p.topk(20, dim=1).indices)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_batches_of_every_size_agree(dt):
    """the row count selects other kernels and the compaction other moves: the same strings but for near ties"""
    model, P = sharp_model(TINY, 12, dt)
    z = torch.randn(17000, TINY["Dz"], generator=torch.Generator().manual_seed(4))
    big = model.beam_search_tokens(z, 4, 30)             # 17000 molecules: two library calls, the first of 16384
    for rows in (slice(0, 1), slice(5, 70), slice(16380, 16390)):
        part = model.beam_search_tokens(z[rows], 4, 30)
        check_scores(P, z[rows].numpy(), part, dt)
        assert bool(((part[0] == big[0][rows]).all(-1).float().mean() > (0.95 if dt == "fp32" else 0.4)))
    check_scores(P, z[16000:16100].numpy(), [t[16000:16100] for t in big], dt)


def test_many_molecules_leave_and_close_up():
    """above 16384 positions in one call (the other compaction path), molecules ending all over"""
    model, P = sharp_model(TINY, 14, "fp32")
    n = 20000
    z = torch.randn(n, TINY["Dz"], generator=torch.Generator().manual_seed(6))
    out = model.beam_search_tokens(z, 2, 40)
    pick = np.r_[0:40, 9990:10030, n - 40:n]
    check_scores(P, z[pick].numpy(), [t[torch.from_numpy(pick).cuda()] for t in out], "fp32")
    last = out[1].max(1).values
    assert (last <= 8).float().mean() > 0.1 and (last == 40).float().mean() > 0.1          # they did leave at different times


def test_operators_driven_from_outside():
    """a program's own decode loop (torch's GRU arithmetic, fp32) over beam_select, reorder_pages, compact_pages and fork_pages
    finds what VAE.beam_search finds"""
    from polygon_amd import vae
    model, P = sharp_model(TINY, 18, "fp32")
    n, K, T, H, L = 40, 6, 25, TINY["Hd"], TINY["L"]
    z = torch.randn(n, TINY["Dz"], generator=torch.Generator().manual_seed(9)).cuda()
    want = [t.cpu() for t in model.beam_search_tokens(z, K, T)]
    w = {k: torch.from_numpy(v).float().cuda() for k, v in P.items()}
    start = z @ w["decoder_lat.weight"].T + w["decoder_lat.bias"]
    planes = [torch.zeros(n * K, H, device="cuda") for _ in range(L)] + [torch.zeros(n * K, T, dtype=torch.uint8, device="cuda")]
    rows = torch.arange(n, dtype=torch.int32, device="cuda").repeat_interleave(K)
    vae.fork_pages(planes[:L], [start] * L, rows)
    zr = z.repeat_interleave(K, 0)
    tok = torch.full((n, K), model.bos, dtype=torch.int32, device="cuda")
    planes[L][:, 0] = model.bos
    scores = torch.full((n, K), -float("inf"), device="cuda")
    scores[:, 0] = 0
    fin = torch.zeros(n, K, dtype=torch.bool, device="cuda")
    mol = torch.arange(n, device="cuda")
    found = {}
    for t in range(1, T):
        x = torch.cat([w["x_emb.weight"][tok.flatten().long()], zr], 1)
        for l in range(L):
            gi = x @ w["decoder_rnn.weight_ih_l%d" % l].T + w["decoder_rnn.bias_ih_l%d" % l]
            gh = planes[l] @ w["decoder_rnn.weight_hh_l%d" % l].T + w["decoder_rnn.bias_hh_l%d" % l]
            r, u = torch.sigmoid(gi[:, :2 * H] + gh[:, :2 * H]).chunk(2, 1)
            new = torch.tanh(gi[:, 2 * H:] + r * gh[:, 2 * H:])
            planes[l].copy_((1 - u) * new + u * planes[l])
            x = planes[l]
        y = x @ w["decoder_fc.weight"].T + w["decoder_fc.bias"]
        step = vae.beam_select(y.view(len(mol), K, -1), scores, fin, eos=model.eos, pad=model.pad, keep_slots=True)
        vae.reorder_pages(planes, step.parents)
        scores, fin, tok = step.scores, step.finished, step.tokens
        planes[L][:, t] = tok.flatten().to(torch.uint8)
        done = fin.all(1) if t + 1 < T else torch.ones_like(fin[:, 0])
        if not done.any():
            continue
        for i in done.nonzero().flatten().tolist():
            found[int(mol[i])] = (planes[L].view(len(mol), K, T)[i].cpu(), scores[i].cpu(), t)
        group = [p.view(len(mol), -1) for p in planes + [zr]]
        extra = [scores, fin, tok, mol.view(-1, 1)]
        count, place = vae.compact_pages(group + extra, ~done)
        m = int(count)
        if m == 0:
            break
        assert m == int((~done).sum()) and torch.equal(place[~done].sort().values.cpu(), torch.arange(m, dtype=torch.int32))
        planes, zr = [g[:m].reshape(m * K, -1) for g in group[:-1]], group[-1][:m].reshape(m * K, -1)
        scores, fin, tok, mol = extra[0][:m], extra[1][:m], extra[2][:m], extra[3][:m, 0]
    assert len(found) == n
    out = [torch.full((n, K, T), model.pad, dtype=torch.uint8), torch.zeros(n, K, dtype=torch.int32), torch.zeros(n, K)]
    same = 0
    for i in range(n):
        tokens, sc, t = found[i]
        order = sc.argsort(descending=True, stable=True)
        out[0][i, :, :t + 1], out[2][i] = tokens[order][:, :t + 1], sc[order]
        for j, row in enumerate(out[0][i].tolist()):
            out[1][i, j] = row.index(model.eos) + 1 if model.eos in row else T
        same += torch.equal(out[0][i], want[0][i])
    check_scores(P, z.cpu().numpy(), out, "fp32")
    assert same >= 0.9 * n       # (the rest: beams that two fp32 evaluations order differently)


def test_stream_and_graph():
    model, P = sharp_model(TINY, 15, "bf16")
    zs = torch.randn(50, TINY["Dz"], generator=torch.Generator().manual_seed(7)).cuda()
    eager = model.beam_search_tokens(zs, 5, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = model.beam_search_tokens(zs, 5, 20)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    z = zs.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.beam_search_tokens(z, 5, 20)
    for k in range(4):
        z.copy_(zs.roll(k, 0) * (1 + 0.1 * k))
        graph.replay()
        want = model.beam_search_tokens(z, 5, 20)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    model, _ = build_model(TINY, 1, "fp32")
    z = torch.randn(3, TINY["Dz"])
    for bad in (dict(beam_width=0), dict(beam_width=33), dict(max_len=1), dict(temp=0.0), dict(temp=float("nan")),
                dict(allowed=torch.ones(5))):
        with pytest.raises(RuntimeError):                # PolygonHipError is one
            model.beam_search(z, **dict(dict(beam_width=4, max_len=9), **bad))
    with pytest.raises(RuntimeError):
        model.beam_search(z[:, :3])
    with pytest.raises(RuntimeError):
        model.beam_search(z[0])
    assert model.beam_search(z[:0], 4, 9)[0] == []
    L, d = _lib.lib(), model._engine.dims
    L.pg_beam_search_workspace_bytes.restype = ctypes.c_size_t
    assert L.pg_beam_search_workspace_bytes(ctypes.byref(d), 0, 0, 4, 9) == 0
    one = torch.empty(1, device="cuda")
    st = L.pg_beam_search(ctypes.byref(d), 0, _lib.ptr(one), _lib.ptr(one), _lib.ptr(one), ctypes.c_size_t(4), 3, 4, 9, _lib.ptr(one), None,
                          ctypes.c_double(1.0), _lib.ptr(one), _lib.ptr(one), _lib.ptr(one), None)
    assert st == -4 and b"workspace" in L.pg_last_error()
