"""Operators of beam search on the device: the selection over beams and vocabulary, and the moves of the decoder states that
follow it (pg_beam_select, pg_pages_reorder, pg_pages_fork, pg_pages_compact of include/polygon_hip.h).  ``VAE.beam_search``
runs the whole decode; these serve a program that drives its own.

All work is enqueued on the current stream of the tensors' device; nothing synchronises or copies to the host.  Arguments are
checked on the host (shapes, types, devices, strides); indices are device data and checked by the kernels: one that is out of
range moves nothing.  Nothing here is differentiable; pages that move are tensors modified in place, and count as that for
autograd: a backward pass that needs what they held raises.
"""
import ctypes
import struct
from typing import NamedTuple

import torch
from torch.autograd.graph import increment_version

from polygon_amd import _lib

MAX_BEAMS = 32      # PG_MAX_BEAMS
NO_WORKSPACE_V = 1024     # up to here pg_beam_select_workspace_bytes is 0: not asked
INT_END = 1 << 31         # the C entries' numbers are 32 bits wide, and ctypes drops what is above them


class BeamStep(NamedTuple):
    """One step of the selection, every member [n, K] and indexed by the place a beam now has."""
    scores: torch.Tensor        # float32: sum of the log-probabilities, -inf where there was no candidate
    parents: torch.Tensor       # int32: the place, before the step, of the beam this one continues
    tokens: torch.Tensor        # int32: the symbol appended to it
    finished: torch.Tensor      # bool


_entry = None


def _entries():
    """The library's entry points with their argument types declared once (ctypes then converts plain ints by itself)."""
    global _entry
    if _entry is None:
        L = _lib.lib()
        i, l, p, z, d = ctypes.c_int, ctypes.c_long, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_double
        L.pg_beam_select.argtypes = [i, p, l, l, i, i, i, p, l, l, d, p, p, i, i, i, p, p, p, p, p, z, p]
        L.pg_beam_select_workspace_bytes.argtypes, L.pg_beam_select_workspace_bytes.restype = [i, i, i, i], z
        L.pg_pages_reorder.argtypes = [p, i, i, i, p, p]
        L.pg_pages_fork.argtypes = [p, p, i, i, i, p, p]
        L.pg_pages_compact.argtypes = [p, i, i, p, p, p, p, z, p]
        L.pg_pages_compact_workspace_bytes.argtypes, L.pg_pages_compact_workspace_bytes.restype = [i], z
        _entry = L
    return _entry


def _call(device, entry, *args):
    """Runs a C entry on ``device``'s current stream (its last argument), with that device current for the length of the call."""
    if device.type != "cuda":
        raise _lib.PolygonHipError("polygon_amd computes only on an MI355X (`cuda`) device, got a tensor on %s" % device)
    at, now = device.index, torch._C._cuda_getDevice()
    if at == now:
        status = entry(*args, torch._C._cuda_getCurrentRawStream(at))
    else:
        with torch.cuda.device(at):
            status = entry(*args, torch._C._cuda_getCurrentRawStream(at))
    if status:
        _lib.check(status, entry.__name__)


def _flags(t, shape, device, what):
    if t.dtype is not torch.bool and t.dtype is not torch.uint8:
        raise ValueError("%s must be bool or uint8, got %s" % (what, t.dtype))
    if t.shape != shape or t.device != device:
        raise ValueError("%s must be %s on %s, got %s on %s" % (what, list(shape), device, list(t.shape), t.device))
    return t.contiguous()


def beam_select(logits, scores, finished=None, mask=None, temp=1.0, eos=-1, pad=0, keep_slots=False) -> BeamStep:
    """The K best of the K * V continuations of every group's K beams.

    ``logits`` [n, K, V] float32 or bfloat16 (any strides; the last dimension is copied if it is not dense), ``scores`` [n, K]
    float32 (-inf: a place without a beam), ``finished`` [n, K] bool (a finished beam competes with its own score and appends
    ``pad``), ``mask`` [V], [K, V], [n, 1, V] or [n, K, V] bool (False: the symbol is left out, also of the normaliser; what
    the logits hold there is not looked at).  A candidate's score is scores + log_softmax(logits / temp) with the normaliser in
    64 bits; equal scores go by the lower k * V + v.  ``eos`` (-1: none) finishes a beam.  K <= 32, V <= 2**20.

    ``keep_slots``: the best child of a beam stays in that beam's place and the others take the places that became free,
    instead of the order by rank: then ``reorder_pages`` moves only the states of beams with more than one child."""
    if logits.dim() != 3 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("logits must be [n, K, V] float32 or bfloat16, got %s %s" % (list(logits.shape), logits.dtype))
    n, K, V = logits.shape
    dev = logits.device
    if scores.shape != (n, K) or scores.dtype != torch.float32 or scores.device != dev:
        raise ValueError("scores must be [%d, %d] float32 on %s, got %s %s on %s" % (n, K, dev, list(scores.shape), scores.dtype,
                                                                                  scores.device))
    if not (-INT_END <= eos < INT_END and -INT_END <= pad < INT_END and n < INT_END and K < INT_END and V < INT_END):
        raise ValueError("n=%d, K=%d, V=%d, eos=%d, pad=%d: not all fit 32 bits" % (n, K, V, eos, pad))
    if V > 1 and logits.stride(2) != 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    if finished is not None:
        finished = _flags(finished, (n, K), dev, "finished")
    mg = mr = 0
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or mask.device != dev:
            raise ValueError("mask must be bool or uint8 on %s, got %s on %s" % (dev, mask.dtype, mask.device))
        if not 1 <= mask.dim() <= 3 or mask.shape[-1] != V \
                or any(a not in (1, b) for a, b in zip(mask.shape[:-1], (n, K)[3 - mask.dim():])):
            raise ValueError("mask %s does not fit logits %s" % (list(mask.shape), list(logits.shape)))
        if V > 1 and mask.stride(-1) != 1:
            mask = mask.contiguous()
        if mask.dim() > 1 and mask.shape[-2] > 1:
            mr = mask.stride(-2)
        if mask.dim() > 2 and mask.shape[0] > 1:
            mg = mask.stride(0)
    L = _entries()
    like = torch.empty_like              # (the quickest way to an output's memory)
    parents = like(scores, dtype=torch.int32)
    out = BeamStep(like(scores), parents, like(parents), like(scores, dtype=torch.bool))
    code = _lib.PG_F32 if logits.dtype == torch.float32 else _lib.PG_BF16
    need = L.pg_beam_select_workspace_bytes(code, n, K, V) if V > NO_WORKSPACE_V else 0
    ws = scores.new_empty(need, dtype=torch.uint8) if need else None
    _call(dev, L.pg_beam_select, code, logits.data_ptr(), logits.stride(0), logits.stride(1), n, K, V,
          None if mask is None else mask.data_ptr(), mg, mr, float(temp), scores.data_ptr(),
          None if finished is None else finished.data_ptr(), int(eos), int(pad), int(bool(keep_slots)),
          *[t.data_ptr() for t in out], None if ws is None else ws.data_ptr(), need)
    return out


def _planes(planes, what):
    """The C description of a cache (pg_plane: base, pitch, bytes - three words a plane): the planes' first dimension counts pages,
    what is behind it is one page's dense row."""
    if not planes:
        raise ValueError("%s: no planes" % what)
    shape, dev = planes[0].shape, planes[0].device
    P = shape[0] if shape else -1
    if P >= INT_END:
        raise ValueError("%s: %d pages, their number does not fit 32 bits" % (what, P))
    out = []
    for t in planes:
        shape = t.shape
        if not shape or shape[0] != P or t.device != dev:
            raise ValueError("%s: every plane must have the same number of pages in front, on one device" % what)
        if t.requires_grad:
            raise ValueError("%s: pages are moved in place, a plane must not require gradients" % what)
        if P and t.is_contiguous():
            row = pitch = t.nbytes // P
        else:
            row = size = t.element_size()
            pitch = t.stride(0) * size
            for extent, stride in zip(reversed(shape[1:]), reversed(t.stride()[1:])):
                if extent != 1 and stride * size != row:
                    raise ValueError("%s: what is behind a plane's first dimension must be dense, got strides %s" % (what, list(t.stride())))
                row *= extent
            if P <= 1:
                pitch = row
        if row == 0:
            raise ValueError("%s: a page of no bytes" % what)
        out += (t.data_ptr(), pitch, row)
    return struct.pack("%dQ" % len(out), *out), dev, P


def _index(t, dev, what):
    if t.dtype is not torch.int32 or t.device != dev:
        raise ValueError("%s must be int32 on %s, got %s on %s" % (what, dev, t.dtype, t.device))
    return t.contiguous()


def reorder_pages(planes, parents):
    """In place: page g*K + j of every plane takes over what page g*K + parents[g, j] held before the call.  ``planes``:
    tensors [n*K, ...], dense behind the first dimension; ``parents`` [n, K] int32 (``BeamStep.parents``), outside the planes."""
    d, dev, P = _planes(planes, "reorder_pages")
    shape = parents.shape
    if len(shape) != 2 or shape[0] * shape[1] != P:
        raise ValueError("parents %s does not name %d pages" % (list(shape), P))
    parents = _index(parents, dev, "parents")
    _call(dev, _entries().pg_pages_reorder, d, len(planes), shape[0], shape[1], parents.data_ptr())
    increment_version(planes)


def fork_pages(dst, src, index):
    """Page i of ``dst`` becomes a copy of page index[i] of ``src`` in every plane (index int32 [n_dst]; a page may be taken any
    number of times; a negative index or one behind the last page leaves page i as it is).  dst shares no memory with src or
    index."""
    d, dev, P = _planes(dst, "fork_pages: dst")
    s, sdev, Q = _planes(src, "fork_pages: src")
    same = len(dst) == len(src) and sdev == dev
    for a, b in zip(dst, src):
        same = same and a.dtype is b.dtype and a.shape[1:] == b.shape[1:]
    if not same:
        raise ValueError("fork_pages: dst and src must have the same planes but for the number of pages")
    if index.shape != (P,):
        raise ValueError("index %s does not name a page for each of %d" % (list(index.shape), P))
    index = _index(index, dev, "index")
    _call(dev, _entries().pg_pages_fork, d, s, len(dst), P, Q, index.data_ptr())
    increment_version(dst)


def compact_pages(planes, live):
    """Frees the pages whose ``live`` flag ([P] bool) is not set and closes the gaps, in place: the live pages behind the new
    end move, in order, to the dead places before it.  Returns (count int32 [1], map int32 [P]: the new place of every old
    page, -1 for a freed one), both on the device.  ``live`` is read while pages move: where the flags are a plane themselves,
    pass a copy."""
    d, dev, P = _planes(planes, "compact_pages")
    live = _flags(live, (P,), dev, "live")
    L = _entries()
    need = L.pg_pages_compact_workspace_bytes(P)
    count = torch.empty(1, device=dev, dtype=torch.int32)
    where, ws = count.new_empty(P), count.new_empty(need, dtype=torch.uint8) if need else None
    _call(dev, L.pg_pages_compact, d, len(planes), P, live.data_ptr(), count.data_ptr(), where.data_ptr(),
          None if ws is None else ws.data_ptr(), need)
    increment_version(planes)
    return count, where
