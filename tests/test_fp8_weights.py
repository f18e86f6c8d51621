"""CPU checks of the weight quantiser on a module's own parameters."""
import pytest
import torch


@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quantised_parameters_carry_no_gradient(dtype, kind):
    """A weight that records gradients, with a norm weight that does: the quantised copy stands alone (a graph would
    keep the fp32 intermediates, several times the weight), and is the detached weight's, bit for bit."""
    from starkv import fp8_quantize_weight
    g = torch.Generator().manual_seed(2)
    linear, norm = torch.nn.Linear(300, 200, bias=False, dtype=dtype), torch.nn.Parameter(torch.rand(300, generator=g).to(dtype))
    with torch.no_grad():
        linear.weight.copy_(torch.randn(200, 300, generator=g))
    scale = torch.float8_e8m0fnu if kind == "e8m0" else torch.float32
    assert torch.is_grad_enabled() and linear.weight.requires_grad
    q, s = fp8_quantize_weight(linear.weight, scale, norm_weight=norm)
    for t in (q, s):
        assert not t.requires_grad and t.grad_fn is None and t.is_leaf
    want = fp8_quantize_weight(linear.weight.detach(), scale, norm_weight=norm.detach())
    assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s.float(), want[1].float())
    assert torch.is_grad_enabled()
