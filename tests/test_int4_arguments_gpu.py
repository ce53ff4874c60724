"""Arguments of the 4-bit operators that must not be taken for others."""
import pytest
import torch

from llama_pure_compute_b200.int4_linear import Int4Weight, int4_linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def test_residual_and_output_have_the_outputs_width():
    """[n, tokens] has as many values as [tokens, n], but others."""
    w = Int4Weight(torch.randn(32, 128, device=DEV).to(BF))
    x = torch.randn(2, 128, device=DEV).to(BF)
    turned = torch.zeros(32, 2, dtype=BF, device=DEV)
    for bad in (turned, turned.view(-1), turned.view(4, 16)):
        with pytest.raises(ValueError, match="residual must be"):
            int4_linear(x, w, "residual", resid=bad)
        with pytest.raises(ValueError, match="out must be"):
            int4_linear(x, w, out=bad)
    y = int4_linear(x, w)
    r = torch.randn(2, 1, 32, device=DEV).to(BF)  # other leading dims of the same rows
    assert torch.equal(int4_linear(x.view(1, 2, 128), w, "residual", resid=r).view(2, 32),
                       int4_linear(x, w, "residual", resid=r.view(2, 32)))
    assert int4_linear(x, w, out=r).shape == r.shape and torch.equal(r.view(2, 32), y)
    one = torch.zeros(32, dtype=BF, device=DEV)
    assert torch.equal(int4_linear(x[0], w, out=one), one) and torch.equal(one, int4_linear(x[:1], w)[0])
