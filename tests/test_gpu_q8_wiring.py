"""The 8-bit cache and key spans on the model's paths: what a wrong wiring would change."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("wants", ["x", "context", "q", "k", "v"])
def test_context_lengths_drop_no_gradient(wants):
    """Whichever of the inputs and weights wants one: the norms in front run outside of autograd on CUDA."""
    from streamdiffusionv2_b200.wan_model import TextCrossAttention
    m = TextCrossAttention(256, 2).to(DEV, torch.bfloat16).requires_grad_(False)
    x, ctx = _randn(1, 1, 4, 256), _randn(2, 1, 5, 256)
    {"x": x, "context": ctx}[wants].requires_grad_() if wants in ("x", "context") else getattr(m, wants).requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        m(x, ctx, [3])
