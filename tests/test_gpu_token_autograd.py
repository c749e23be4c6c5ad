"""The 8-bit token calls and the layers over them under the tracer: what it cannot follow is handed to a Function, or refused."""
import pytest
import torch
import torch.nn as nn

from actnn_amd import layers
from actnn_amd.conf import config
from actnn_amd.cpp_extension import backward_func as bf
from actnn_amd.cpp_extension import tokens

DEV = "cuda:0"


@pytest.fixture(autouse=True)
def fresh_config():
    config.reset()
    yield
    config.reset()


class Answering(nn.Module):
    """Group norm + SiLU over channels, then a linear layer over the channels of each pixel."""

    def __init__(self):
        super().__init__()
        self.norm, self.act, self.out = layers.QGroupNorm(4, 64), nn.SiLU(), layers.QInt8Linear(64, 40)

    def forward(self, x):
        return self.out(layers.gn_silu(self.norm, self.act, x).permute(0, 2, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode, torch.enable_grad])
@pytest.mark.parametrize("held", [False, True])
def test_a_traced_model_answers_like_the_model(mode, held):
    torch.manual_seed(1)
    model = Answering().to(DEV).eval()
    with mode():
        if held:
            model.out.hold_weight()
        traced = torch.jit.trace(model, torch.randn(2, 64, 9, device=DEV))
        for shape in ((2, 64, 9), (3, 64, 5)):
            x = torch.randn(shape, device=DEV)
            got = traced(x)
            assert torch.equal(got, model(x))
        x = torch.randn(2, 9, 64, device=DEV).permute(0, 2, 1)               # channels last already
        got = traced(x)
        assert torch.equal(got, model(x))


def test_calls_by_themselves_are_not_traced():
    # (the refusal comes before anything is asked of the tensors)
    q, s, x = torch.zeros(4, 16, dtype=torch.int8), torch.ones(4), torch.zeros(4, 16)
    m = torch.zeros(4, 2)
    for call in (lambda x: tokens.quantize_tokens(x), lambda x: tokens.dequantize_tokens(q, x[:, 0]),
                 lambda x: tokens.matmul_tokens(q, x[:, 0], q, s), lambda x: tokens.linear_tokens(x, q, s),
                 lambda x: tokens.linear_tokens_grad_weight(x, q, s),
                 lambda x: bf.hip_group_norm_forward(x, 2, None, None, 1e-5)[0],
                 lambda x: bf.hip_group_norm_backward(x, None, None, 2, None, None, m, m, input=x)[0]):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, x)
