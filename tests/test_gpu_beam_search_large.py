"""pg_beam_search called for more latents than the cells' operands reach at once (2 GiB of states, 65535 tiles of 64 rows): it gives
what calls of a few ten thousand rows give, bit for bit - every row's arithmetic is its own."""
import ctypes

import numpy as np
import pytest
import torch

from polygon_amd import _lib
from tests.helpers import REAL, TINY, build_model
from tests.test_gpu_beam_search import check_scores

pytestmark = pytest.mark.gpu


def one_call(model, z, K, max_len):
    """the C entry for all latents at once, where beam_search_tokens cuts at 65536 rows"""
    eng, L, n = model._engine, _lib.lib(), z.shape[0]
    eng.ensure_shadow()
    L.pg_beam_search_workspace_bytes.restype = ctypes.c_size_t
    need = L.pg_beam_search_workspace_bytes(ctypes.byref(eng.dims), eng.dtype_code(), n, K, max_len)
    assert need > 0, L.pg_last_error()
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = (torch.full((n, K, max_len), 255, dtype=torch.uint8, device="cuda"), torch.full((n, K), -1, dtype=torch.int32, device="cuda"),
           torch.full((n, K), 1.0, device="cuda"))
    _lib.check(L.pg_beam_search(ctypes.byref(eng.dims), eng.dtype_code(), _lib.ptr(eng.flat), _lib.ptr(eng.shadow), _lib.ptr(ws),
                                ctypes.c_size_t(need), n, K, max_len, _lib.ptr(z), None, ctypes.c_double(1.0), *[_lib.ptr(t) for t in out],
                                _lib.stream_ptr()), "pg_beam_search")
    return out


@pytest.mark.parametrize("dims,dt,n,K,max_len", [(REAL, "fp32", 557100, 2, 3), (TINY, "bf16", 133200, 32, 12), (TINY, "fp32", 133200, 32, 12)])
def test_more_rows_than_the_cells_reach(dims, dt, n, K, max_len):
    model, P = build_model(dims, 17, dt, eos_bias=2.0)
    z = torch.randn(n, dims["Dz"], generator=torch.Generator().manual_seed(8)).cuda()
    got = one_call(model, z, K, max_len)
    want = model.beam_search_tokens(z, K, max_len)
    part = 65536 // K
    same = n // part * part            # (behind it the wrapper's last call has few rows: other kernels)
    for a, b in zip(got, want):
        assert torch.equal(a[:same], b[:same])
    pick = np.r_[0:8, n // 2 - 8:n // 2 + 8, n - 8:n]
    rows = torch.from_numpy(pick).cuda()
    check_scores(P, z[rows].cpu().numpy(), [t[rows] for t in got], dt)
