"""What pg_beam_search does on the host, before any launch.  No GPU needed."""
import ctypes

import pytest

from polygon_amd import _lib
from polygon_amd.vae.vae_model import _Dims

DESCRIPTOR = 1 << 31        # the cells read their operands by 32-bit offsets that end below this many bytes
GRID = 65535 * 64           # rows that one launch of the cells' 64-row tiles takes


def _bytes(d, dtype, n, K, max_len=3):
    L = _lib.lib()
    L.pg_beam_search_workspace_bytes.restype = ctypes.c_size_t
    return L.pg_beam_search_workspace_bytes(ctypes.byref(d), dtype, n, K, max_len)


def _dims(Hd, Dz, L=3):
    return _Dims(V=51, E=51, Hq=32, Dz=Dz, Hd=Hd, L=L, pad=0, bos=1, eos=2, unk=3, Lq=1, qbidir=0)


@pytest.mark.parametrize("dtype,es", [(_lib.PG_F32, 4), (_lib.PG_BF16, 2)])
@pytest.mark.parametrize("Hd,Dz,K", [(512, 128, 1), (512, 128, 8), (64, 16, 32), (32, 8, 1), (2048, 64, 32), (32, 8192, 3)])
def test_latents_beyond_the_cells_reach_are_taken_in_turn(Hd, Dz, K, dtype, es):
    """every latent of a call is decoded by arrays that the cells and the products can address: a call of more latents than that
    reuses the workspace of as many as can go together"""
    d = _dims(Hd, Dz)
    most = min((DESCRIPTOR - 1) // (max(K * Hd, Dz) * es), GRID // K)
    whole = _bytes(d, dtype, most, K)
    assert whole > 0
    n_max = ((1 << 24) - 1) // K
    for n in (most + 1, 2 * most, 2 * most + 1, 5 * most + 3, n_max):
        if n > n_max:
            continue
        turns = -(-n // most)
        assert 0 < _bytes(d, dtype, n, K) <= whole
        assert _bytes(d, dtype, n, K) == _bytes(d, dtype, -(-n // turns), K)      # turns of one size
    assert _bytes(d, dtype, n_max + 1, K) == 0


def test_a_latent_that_no_call_could_decode_is_refused():
    assert _bytes(_dims(1 << 24, 8, L=1), _lib.PG_F32, 1, 32) == 0 and b"2 GiB" in _lib.lib().pg_last_error()
    assert _bytes(_dims(1 << 20, 8, L=1), _lib.PG_F32, 1, 32) > 0


def test_search_checks_its_numbers_before_anything_is_allocated():
    """(a max_len that 32 bits do not hold would fill its tensors' first columns only)"""
    import torch
    from polygon_amd.vae.vae_model import VAE
    model, z = VAE(q_d_h=32, d_z=16, d_d_h=32, d_n_layers=1), torch.zeros(0, 16)
    for max_len in ((1 << 32) + 5, (1 << 20) + 1, 1, -3):
        with pytest.raises(RuntimeError, match="max_len"):
            model.beam_search_tokens(z, 4, max_len)
    for width in (0, 33, (1 << 32) + 1):
        with pytest.raises(RuntimeError, match="beam_width"):
            model.beam_search_tokens(z, width, 9)
