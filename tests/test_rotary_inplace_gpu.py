"""Rotation in place of rows that an autograd graph has kept."""
import pytest
import torch

from llm_inference_optimization_b200 import rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["q", "k"])
def test_a_graph_that_kept_the_rows_notices(cuda_device, which):
    """The backward pass of an earlier product needs the rows as they were: it is refused and gives no wrong gradient."""
    r = rotary.RotaryEmbedding(64, device=cuda_device)
    pos = torch.arange(1, 6, dtype=torch.int32, device=cuda_device)
    w = torch.randn(5, 2, 64, device=cuda_device, requires_grad=True)
    kept = w * 2
    loss = (kept * kept).sum()
    other = torch.randn(5, 2, 64, device=cuda_device)
    with torch.no_grad():
        r.apply(pos, *((kept, other) if which == "q" else (other, kept)), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                     # tensors without versions
        x = torch.randn(5, 2, 64, device=cuda_device)
        want = r.apply(pos, x)
        assert torch.equal(r.apply(pos, x, inplace=True), want)


def test_out_of_place_leaves_the_graph_alone(cuda_device):
    r = rotary.RotaryEmbedding(64, device=cuda_device)
    pos = torch.arange(1, 6, dtype=torch.int32, device=cuda_device)
    w = torch.randn(5, 2, 64, device=cuda_device, requires_grad=True)
    kept = w * 2
    loss = (kept * kept).sum()
    with torch.no_grad():
        r.apply(pos, kept)
    loss.backward()
    assert torch.allclose(w.grad, 8 * w.detach())
