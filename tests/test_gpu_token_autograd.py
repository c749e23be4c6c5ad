"""The 8-bit token calls and the layers over them under the tracer, in forward mode and in reverse mode: what these cannot follow
is handed to a Function that they can, or refused."""
import pytest
import torch
import torch.autograd.forward_ad as fwad
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


def operands():
    """Every call with its differentiable arguments: name -> (function of them, the arguments)."""
    torch.manual_seed(2)
    x, w, b = torch.randn(6, 32, device=DEV), torch.randn(8, 32, device=DEV), torch.randn(8, device=DEV)
    c, s = tokens.quantize_tokens(x)
    wc, ws = tokens.quantize_tokens(w)
    g = torch.randn(6, 8, device=DEV).half()
    a, d = torch.rand(32, device=DEV) + 0.5, torch.randn(32, device=DEV)
    y, mean, rstd, codes, scale = bf.hip_group_norm_forward(x, 4, a, d, 1e-5, "silu", keep=True)
    return {
        "quantize_tokens": (lambda x: tokens.quantize_tokens(x)[1], (x,)),
        "dequantize_tokens": (lambda s: tokens.dequantize_tokens(c, s), (s,)),
        "matmul_tokens": (lambda s, ws, b: tokens.matmul_tokens(c, s, wc, ws, b), (s, ws, b)),
        "linear_tokens": (lambda x, ws, b: tokens.linear_tokens(x, wc, ws, b), (x, ws, b)),
        "linear_tokens, kept": (lambda x, ws, b: tokens.linear_tokens(x, wc, ws, b, keep=True)[0], (x, ws, b)),
        "linear_tokens_grad_weight": (lambda g, s: tokens.linear_tokens_grad_weight(g, c, s), (g, s)),
        "group_norm_forward": (lambda x, a, d: bf.hip_group_norm_forward(x, 4, a, d, 1e-5, "silu")[0], (x, a, d)),
        "group_norm_backward": (lambda y, a, d, m, r: bf.hip_group_norm_backward(y, codes, scale, 4, a, d, m, r, "silu")[0],
                                (y, a, d, mean, rstd)),
    }


@pytest.mark.gpu
def test_tangents_are_refused():
    for name, (call, given) in operands().items():
        for i in range(len(given)):
            with fwad.dual_level(), torch.no_grad():
                args = list(given)
                args[i] = fwad.make_dual(given[i], torch.ones_like(given[i]))
                with pytest.raises(RuntimeError, match="forward"):
                    call(*args)
            assert torch.equal(call(*given), call(*given)), name          # and nothing of it stays


@pytest.mark.gpu
@pytest.mark.parametrize("frozen", [False, True])
def test_tangents_are_refused_by_the_layers(frozen):
    for layer in (layers.QInt8Linear(32, 8).to(DEV), layers.QGroupNorm(4, 32).to(DEV)):
        layer.requires_grad_(not frozen)
        x = torch.randn(6, 32, device=DEV)
        for grad in (True, False):
            with fwad.dual_level(), torch.set_grad_enabled(grad):
                with pytest.raises(RuntimeError, match="forward"):
                    layer(fwad.make_dual(x, torch.ones_like(x)))


@pytest.mark.gpu
def test_calls_without_a_derivative_say_so_in_the_backward_pass():
    for name, (call, given) in operands().items():
        want = call(*given)
        for i in range(len(given)):
            args = list(given)
            args[i] = given[i].clone().requires_grad_()
            y = call(*args)
            assert torch.equal(y.detach(), want) and y.requires_grad, name
            with pytest.raises(RuntimeError, match=f"derivative for {name.split(',')[0]} is not implemented"):
                y.float().sum().backward()
            assert args[i].grad is None
            with torch.no_grad():
                assert not call(*args).requires_grad
        assert not call(*given).requires_grad


@pytest.mark.gpu
def test_a_result_cut_out_of_a_larger_one_says_so_too():
    # (a gradient of odd width whose product runs over whole chunks)
    c, s = tokens.quantize_tokens(torch.randn(1156, 1728, device=DEV))
    g = torch.randn(1156, 673, device=DEV).bfloat16()
    want = tokens.linear_tokens_grad_weight(g, c, s)
    got = tokens.linear_tokens_grad_weight(g.requires_grad_(), c, s)
    assert torch.equal(got.detach(), want)
    with pytest.raises(RuntimeError, match="derivative for linear_tokens_grad_weight is not implemented"):
        got.float().sum().backward()
