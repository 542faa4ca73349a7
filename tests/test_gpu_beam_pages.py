"""Moves of pages between planes of one buffer, and what autograd hears of moves in place."""
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


@pytest.mark.parametrize("how", ["reorder", "fork", "compact"])
def test_autograd_hears_of_moves(how):
    """a plane that was saved for another tensor's gradient and then moved: backward refuses, as after torch's own in-place operators"""
    state, w = torch.randn(6, 64, device="cuda"), torch.randn(64, 64, device="cuda", requires_grad=True)
    view, rest = state[:, :32], torch.randn(6, 32, device="cuda")
    loss = (state @ w).sum()
    before = state._version
    if how == "reorder":
        vae.reorder_pages([rest, view], ints(1, 0, 2, 0, 1, 2).view(2, 3))
    elif how == "fork":
        vae.fork_pages([view], [rest], ints(0, 1, -1, 2, 2, 5))
    else:
        vae.compact_pages([rest, view], torch.tensor([0, 1, 1, 0, 1, 1], dtype=torch.bool, device="cuda"))
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # what a move only reads is not modified
    source, index = torch.randn(6, 64, device="cuda"), ints(0, 0, 1, 1, 2, 5)
    loss = (source @ w).sum()
    vae.fork_pages([torch.empty_like(source)], [source], index)
    loss.backward()
    assert source._version == index._version == 0 and w.grad is not None


def test_moves_of_inference_tensors():
    with torch.inference_mode():
        state = torch.randn(4, 40, device="cuda")
        old = state.clone()
        vae.reorder_pages([state], ints(1, 0, 3, 2).view(1, 4))
        assert torch.equal(state, old[[1, 0, 3, 2]])
        vae.fork_pages([state], [old], ints(0, 1, 2, 3))
        count, _ = vae.compact_pages([state], torch.tensor([False, True, False, True], device="cuda"))
        assert count.item() == 2 and torch.equal(state[:2], old[[3, 1]])
    vae.reorder_pages([state], ints(0, 1, 2, 3).view(1, 4))          # outside of it too
