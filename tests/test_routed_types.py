"""A routed MLP inside a model that is brought to another type: what decides stays in fp32."""
import pytest
import torch

from qmoe_amd import routing, sub1


def routed(bias, experts=4, d_model=8):
    stack = sub1.Sub1Experts.__new__(sub1.Sub1Experts)      # (making one takes a GPU)
    torch.nn.Module.__init__(stack)
    stack._wi, stack._d_model = [None] * experts, d_model
    return routing.RoutedMLP(torch.nn.Linear(d_model, experts), stack, 2, bias=bias)


@pytest.mark.parametrize('change', [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.bfloat16().float()])
def test_the_bias_keeps_its_type_and_values(change):
    bias = torch.tensor([0.1, 1 + 2.0 ** -20, -3.0, 1e-30])
    model = torch.nn.Sequential(routed(bias.clone()), routed(None))
    change(model)
    assert model[0].bias.dtype == torch.float32 and torch.equal(model[0].bias, bias) and model[1].bias is None
    assert dict(model.named_buffers())['0.bias'] is model[0].bias and list(model[0].state_dict())[0] == 'bias'


def test_the_bias_is_moved_and_loaded_as_any_buffer():
    model = routed(torch.ones(4))
    model.to('meta', torch.bfloat16)
    assert model.bias.device.type == 'meta' and model.bias.dtype == torch.float32
    model = routed(torch.ones(4)).bfloat16()
    state = {k: v.bfloat16() for k, v in routed(torch.full((4,), 2.0)).state_dict().items()}
    model.load_state_dict(state)
    assert model.bias.dtype == torch.float32 and bool((model.bias == 2).all())


@pytest.mark.gpu
def test_a_model_in_bf16_routes_as_before():
    from test_gpu_block import block
    *_, routed_mlp, _ = block(64, 96, 8, 3)
    hidden = torch.randn((5, 64), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    want = routed_mlp(hidden)
    for model in (torch.nn.Sequential(routed_mlp).to(torch.bfloat16), torch.nn.Sequential(routed_mlp).cuda()):
        assert all(torch.equal(a, b) for a, b in zip(model[0](hidden), want))
