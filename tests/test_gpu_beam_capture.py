"""VAE.beam_search captured into a graph: the weights' operand copies are laid out before, never inside."""
import pytest
import torch

from polygon_amd._lib import PolygonHipError
from tests.helpers import TINY, build_model

pytestmark = pytest.mark.gpu


def capture(model, z):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.beam_search_tokens(z, 4, 12)
    return graph, out


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_weights_are_not_laid_out_by_a_graph(dt):
    """a capture records launches and runs none: operand copies that it laid out would be missing until a replay, and laid out again
    by each.  A search whose weights are new, changed or moved since the last call refuses to be captured, and is as before
    afterwards."""
    model, _ = build_model(TINY, 19, dt, eos_bias=2.0)
    twin, _ = build_model(TINY, 19, dt, eos_bias=2.0)
    z = torch.randn(9, TINY["Dz"], generator=torch.Generator().manual_seed(3)).cuda()
    with pytest.raises(PolygonHipError, match="captur"):
        capture(model, z)                                    # never called before
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    want = twin.beam_search_tokens(z, 4, 12)
    assert same(model.beam_search_tokens(z, 4, 12), want)
    graph, out = capture(model, z)
    assert same(model.beam_search_tokens(z, 4, 12), want)
    for _ in range(3):
        out[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want)
    with torch.no_grad():
        for m in (model, twin):
            m.decoder_fc.weight.mul_(3.0)
    with pytest.raises(PolygonHipError, match="captur"):
        capture(model, z)                                    # changed
    assert same(model.beam_search_tokens(z, 4, 12), twin.beam_search_tokens(z, 4, 12))
    model.load_state_dict({k: v.clone() for k, v in model.state_dict().items()})
    p = model.decoder_lat.weight
    p.data = p.data.clone()                                  # the same values at another address
    with pytest.raises(PolygonHipError, match="captur"):
        capture(model, z)
    assert same(model.beam_search_tokens(z, 4, 12), twin.beam_search_tokens(z, 4, 12))
    graph, out = capture(model, z)
    graph.replay()
    torch.cuda.synchronize()
    assert same(out, twin.beam_search_tokens(z, 4, 12))
