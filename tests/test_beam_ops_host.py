"""Refusals of the beam-search operators: what the C entries and the Python wrappers turn down on the host, before any kernel
could see it.  No GPU needed."""
import ctypes
import os

import pytest
import torch

from polygon_amd import _lib, vae
from polygon_amd.vae import beam

FAKE = 1 << 20        # an address that nothing reads: every call below ends at its checks


def _select(**kw):
    a = dict(dtype=_lib.PG_F32, logits=FAKE, ld_group=8, ld_row=4, n=1, K=2, V=4, mask=None, mask_group=0, mask_row=0, temp=1.0,
             scores=FAKE, finished=None, eos=-1, pad=0, keep=0, scores_out=FAKE, parents=FAKE, tokens=FAKE, finished_out=FAKE,
             ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return beam._entries().pg_beam_select(*a.values())


@pytest.mark.parametrize("kw", [
    dict(dtype=7), dict(n=-1), dict(K=0), dict(K=33), dict(V=0), dict(V=(1 << 20) + 1), dict(temp=0.0), dict(temp=-1.0),
    dict(temp=float("nan")), dict(temp=float("inf")), dict(temp=1e-320), dict(pad=-1), dict(pad=4), dict(eos=4), dict(logits=None),
    dict(scores=None), dict(scores_out=None), dict(parents=None), dict(tokens=None), dict(finished_out=None)])
def test_select_refuses(kw):
    assert _select(**kw) == -1
    assert b"pg_beam_select" in _lib.lib().pg_last_error()


def test_select_of_no_group_is_nothing():
    assert _select(n=0, logits=None, scores=None) == 0


def _pl(*rows):
    """pg_plane[]: base, pitch, bytes - three words each"""
    flat = [w or 0 for row in rows for w in row]
    return (ctypes.c_long * len(flat))(*flat)


ONE = (FAKE, 64, 64)


def test_pages_refuse():
    L = beam._entries()
    reorder = lambda rows, n=2, K=2, par=FAKE, np=None: L.pg_pages_reorder(_pl(*rows), len(rows) if np is None else np, n, K, par, None)  # noqa: E731
    assert reorder([ONE], n=-1) == reorder([ONE], K=0) == reorder([ONE], K=33) == reorder([ONE], par=None) == -1
    assert reorder([ONE], np=0) == reorder([ONE], np=33) == L.pg_pages_reorder(None, 1, 2, 2, FAKE, None) == -1
    assert reorder([(None, 64, 64)]) == reorder([(FAKE, 63, 64)]) == reorder([(FAKE, 64, 0)]) == -1
    assert reorder([ONE, ONE]) == -1 and b"share" in L.pg_last_error()
    assert reorder([ONE, (FAKE + 32, 64, 64)]) == -1
    assert reorder([(FAKE, 128, 64), (FAKE + 63, 128, 64)]) == -1          # interleaved, one byte in common
    assert reorder([(FAKE, 128, 64), (FAKE + 64, 128, 65)]) == -1          # runs into the next row of the first
    assert reorder([ONE], n=0, par=None) == 0

    fork = lambda d, s, nd=4, ns=4, idx=FAKE: L.pg_pages_fork(_pl(d), _pl(s), 1, nd, ns, idx, None)  # noqa: E731
    far = (FAKE + (1 << 16), 64, 64)
    assert fork(ONE, ONE) == fork(ONE, (FAKE + 192, 64, 64)) == -1         # the last page of dst is the first of src
    assert fork(ONE, (FAKE + (1 << 16), 64, 32)) == fork(ONE, (FAKE + (1 << 16), 16, 64)) == fork(ONE, (None, 64, 64)) == -1
    assert fork(ONE, far, nd=-1) == fork(ONE, far, ns=-1) == fork(ONE, far, idx=None) == -1
    assert L.pg_pages_fork(_pl(ONE), None, 1, 4, 4, FAKE, None) == -1
    assert fork(ONE, far, nd=0, idx=None) == fork(ONE, far, ns=0, idx=None) == 0

    many = 1 << 20
    need = L.pg_pages_compact_workspace_bytes(many)
    compact = lambda n=many, live=FAKE, count=FAKE, m=FAKE, ws=FAKE, size=need: L.pg_pages_compact(_pl((FAKE, 64, 64)), 1, n, live, count, m, ws, size, None)  # noqa: E731
    assert compact(n=-1) == compact(live=None) == compact(count=None) == compact(m=None) == -1
    assert need > 0 and compact(ws=None) == compact(size=need - 1) == -4


def test_indices_are_no_pages():
    """flags, parents and indices that lie inside pages that the call moves would change under the workgroups that read them"""
    L = beam._entries()
    planes, other = _pl((FAKE + (1 << 16), 128, 64), ONE), _pl((FAKE + (1 << 17), 128, 64), (FAKE + (1 << 18), 64, 64))
    refused = lambda status: status == -1 and b"share" in L.pg_last_error()  # noqa: E731
    for at in (FAKE, FAKE + 255, FAKE - 3, FAKE + (1 << 16) + 130, FAKE + (1 << 16) + 60, FAKE + (1 << 16) + 125):
        assert refused(L.pg_pages_reorder(planes, 2, 2, 2, at, None))
        assert refused(L.pg_pages_fork(planes, other, 2, 4, 4, at, None))
        away = FAKE + (1 << 20)
        for args in ((at, away, away + 64), (away, at, away + 64), (away, away + 64, at), (away, away + 3, away + 64), (away, away + 64, away - 15)):
            assert refused(L.pg_pages_compact(planes, 2, 4, *args, None, 0, None))
    assert refused(L.pg_pages_compact(_pl((FAKE, 64, 64)), 1, 1 << 15, FAKE << 4, FAKE << 5, FAKE << 6, FAKE + 640, 1 << 30, None))


def test_interleaved_planes_are_told_from_shared_ones():
    """planes of one buffer: columns [0, 64) and [64, 128) of rows of 128 bytes share nothing, whichever comes first"""
    L = beam._entries()
    a, b = (FAKE, 128, 64), (FAKE + 64, 128, 64)
    assert L.pg_pages_fork(_pl(a), _pl(b), 1, 0, 4, None, None) == 0
    for d, s in ((a, b), (b, a)):      # passes the planes' checks and stops at the missing index
        assert L.pg_pages_fork(_pl(d), _pl(s), 1, 4, 4, None, None) == -1 and b"index" in L.pg_last_error()


def test_wrappers_refuse():
    x, s = torch.zeros(2, 3, 5), torch.zeros(2, 3)
    with pytest.raises(_lib.PolygonHipError):
        vae.beam_select(x, s)                                              # not on the GPU
    for bad in (dict(logits=x[0]), dict(logits=x.double()), dict(logits=x.half()), dict(scores=s[:1]), dict(scores=s.double())):
        with pytest.raises(ValueError):
            vae.beam_select(**dict(dict(logits=x, scores=s), **bad))
    pages, par = torch.zeros(6, 4), torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(_lib.PolygonHipError):
        vae.reorder_pages([pages], par)
    for planes, parents in (([], par), ([pages[:5]], par), ([pages.t()], par[:, :2]), ([pages, pages[:5]], par), ([pages], par.long()),
                            ([pages], par.reshape(-1)), ([pages.clone().requires_grad_()], par), ([torch.zeros(6, 0)], par),
                            ([torch.zeros(6, 4, 4).transpose(1, 2)], par), ([torch.tensor(1.0)], par)):
        with pytest.raises(ValueError):
            vae.reorder_pages(planes, parents)
    idx = torch.zeros(6, dtype=torch.int32)
    for dst, src, index in (([pages], [pages[:, :3]], idx), ([pages], [pages.double()], idx), ([pages], [pages, pages], idx),
                            ([pages], [pages], idx[:5]), ([pages], [pages], idx.long())):
        with pytest.raises(ValueError):
            vae.fork_pages(dst, src, index)
    for live in (torch.zeros(5, dtype=torch.bool), torch.zeros(6)):
        with pytest.raises(ValueError):
            vae.compact_pages([pages], live)


def test_workspace():
    need = beam._entries().pg_beam_select_workspace_bytes
    assert all(need(t, n, K, beam.NO_WORKSPACE_V) == 0 for t in (0, 1) for n in (1, 10 ** 5) for K in (1, 32))
    assert need(0, 1, 1, beam.NO_WORKSPACE_V + 1) > 0 and need(0, 0, 4, 9000) == 0
    assert _select(V=9000, ws=FAKE, ws_bytes=need(0, 1, 2, 9000) - 1) == -4 and _select(V=9000, ws=None, ws_bytes=1 << 20) == -4
    assert _select(n=1 << 20, K=16) == -1                # n * K not below 2^24


def test_limits_match_the_header():
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "polygon_hip.h")).read()
    assert "#define PG_MAX_BEAMS %d\n" % beam.MAX_BEAMS in text and ctypes.sizeof(ctypes.c_long) == ctypes.sizeof(ctypes.c_void_p) == 8


def _bytes_of(plane, pages):
    base, pitch, width = plane
    return {base + p * pitch + i for p in range(pages) for i in range(width)}


def test_planes_of_different_pitches_are_told_from_shared_ones():
    """columns of one buffer by rows, by every other row, or one row alone: refused where bytes are shared, and only there"""
    L = beam._entries()
    at = lambda row, col, step, width: (FAKE + row * 128 + col, step * 128, width)  # noqa: E731
    one = lambda row, col, width: (FAKE + row * 128 + col, width, width)            # noqa: E731  (one page: the pitch says nothing)
    apart = [(one(3, 64, 64), 1, at(0, 0, 1, 64), 8), (one(0, 64, 64), 1, at(0, 0, 1, 64), 8), (one(7, 0, 64), 1, at(0, 64, 1, 64), 8),
             (one(3, 64, 16), 1, one(3, 0, 64), 1), (at(0, 64, 2, 64), 4, at(0, 0, 1, 64), 8), (at(0, 0, 2, 128), 4, at(1, 0, 2, 128), 4),
             (at(0, 0, 2, 128), 4, at(1, 0, 4, 128), 2), (one(9, 0, 64), 1, at(0, 0, 1, 128), 8), (at(1, 32, 3, 32), 3, at(0, 64, 2, 64), 5)]
    shared = [(one(3, 32, 64), 1, at(0, 0, 1, 64), 8), (one(3, 64, 65), 1, at(0, 0, 1, 64), 8), (one(3, 0, 64), 1, one(3, 63, 64), 1),
              (at(0, 32, 2, 64), 4, at(0, 0, 1, 64), 8), (at(0, 0, 2, 128), 4, at(0, 0, 4, 128), 2), (at(1, 60, 3, 32), 3, at(0, 64, 2, 64), 5)]
    for case, share in [(c, False) for c in apart] + [(c, True) for c in shared]:
        a, na, b, nb = case
        assert bool(_bytes_of(a, na) & _bytes_of(b, nb)) == share
        for (d, nd), (s, ns) in (((a, na), (b, nb)), ((b, nb), (a, na))):
            d, s = (d[0], d[1], min(d[2], s[2])), (s[0], s[1], min(d[2], s[2]))       # (a fork's planes have one width)
            if bool(_bytes_of(d, nd) & _bytes_of(s, ns)) != share:
                continue
            assert L.pg_pages_fork(_pl(d), _pl(s), 1, nd, ns, None, None) == -1       # refused, or stops at the missing index
            assert (b"share" if share else b"index is NULL") in L.pg_last_error(), case


def test_planes_share_no_byte_by_counting():
    """random planes: what shares a byte is always refused, whatever the pitches"""
    import random
    rng, L = random.Random(4), beam._entries()
    refused = taken = 0
    for _ in range(4000):
        width = rng.randint(1, 40)
        planes = []
        for _ in range(2):
            n = rng.choice([1, 1, 2, 3, 7])
            planes.append(((FAKE + rng.randint(0, 200), max(width, rng.choice([16, 32, 48, 64, 96, 128, width, width + 5])), width), n))
        (d, nd), (s, ns) = planes
        status = L.pg_pages_fork(_pl(d), _pl(s), 1, nd, ns, None, None)
        assert status == -1
        if _bytes_of(d, nd) & _bytes_of(s, ns):
            assert b"share" in L.pg_last_error()
            refused += 1
        else:
            taken += b"index is NULL" in L.pg_last_error()
    assert refused > 500 and taken > 500


def test_wrappers_refuse_what_the_entries_integers_do_not_hold():
    """the C entries count in 32 bits: a larger number must not reach them as what is left of it"""
    x, s = torch.zeros(2, 3, 5), torch.zeros(2, 3)
    for kw in (dict(eos=1 << 32), dict(eos=-(1 << 32) + 2), dict(pad=1 << 32), dict(pad=(1 << 32) + 1)):
        with pytest.raises(ValueError, match="32 bits"):
            vae.beam_select(x, s, **kw)
    meta = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="meta")  # noqa: E731
    many = (1 << 32) + 1
    for n, K, V in ((many, 1, 1), (1, many, 1), (1, 1, many)):
        with pytest.raises(ValueError, match="32 bits"):
            vae.beam_select(meta(n, K, V), meta(n, K))
    pages, index = meta(many, 4), meta(many, dtype=torch.int32)
    with pytest.raises(ValueError, match="32 bits"):
        vae.reorder_pages([pages], index.view(many, 1))
    with pytest.raises(ValueError, match="32 bits"):
        vae.fork_pages([pages], [meta(3, 4)], index)
    with pytest.raises(ValueError, match="32 bits"):
        vae.fork_pages([meta(3, 4)], [pages], meta(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="32 bits"):
        vae.compact_pages([pages], meta(many, dtype=torch.bool))
