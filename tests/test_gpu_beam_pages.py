"""Moves of pages between planes of one buffer."""
import pytest
import torch

from polygon_amd import vae
from polygon_amd._lib import PolygonHipError

pytestmark = pytest.mark.gpu


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_pages_of_one_buffer_at_other_pitches():
    """one page of a buffer from the columns beside it, and every other row from the rows between"""
    buf = torch.randint(0, 255, (8, 128), dtype=torch.uint8, device="cuda")
    old = buf.clone()
    vae.fork_pages([buf[3:4, 64:]], [buf[:, :64]], ints(5))
    old[3, 64:] = old[5, :64]
    assert torch.equal(buf, old)
    vae.fork_pages([buf[::2]], [buf[1::4]], ints(1, 0, -1, 1))
    old[0], old[2], old[6] = old[5], old[1], old[5]
    assert torch.equal(buf, old)
    vae.fork_pages([buf[:, 100:]], [buf[2:3, 40:68]], ints(*[0] * 8))
    old[:, 100:] = old[2, 40:68]
    assert torch.equal(buf, old)
    for dst, src, index in ((buf[3:4, 32:96], buf[:, :64], ints(0)), (buf[::2], buf[::4], ints(0, 0, 0, 0))):
        with pytest.raises(PolygonHipError):
            vae.fork_pages([dst], [src], index)
    assert torch.equal(buf, old)
