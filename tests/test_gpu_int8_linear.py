"""QInt8Linear in the ways that a model uses it beside plain training: under autocast, frozen, held, without compression."""
import copy

import pytest
import torch
import torch.nn as nn

from actnn_amd import layers
from actnn_amd.conf import config
from actnn_amd.cpp_extension import tokens
from actnn_amd.utils import to_channels_last

DEV = "cuda:0"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def fresh_config():
    config.reset()
    yield
    config.reset()


def allocated(f):
    """What f() returns, and the bytes that live after it and did not before."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = f()
    torch.cuda.synchronize()
    return out, torch.cuda.memory_allocated() - before


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [3, 200])
def test_training_and_answering_multiply_the_same_integers_under_autocast(M, dtype):
    torch.manual_seed(1)
    layer = layers.QInt8Linear(128, 48).to(DEV)
    x = torch.randn(M, 128, device=DEV, requires_grad=True)
    go = torch.randn(M, 48, device=DEV).to(dtype)
    with torch.autocast("cuda", dtype=dtype):
        y = layer(x)
        with torch.no_grad():
            answer = layer(x)
            held = copy.deepcopy(layer).hold_weight()(x)
    assert y.dtype == answer.dtype == dtype and torch.equal(y, answer) and torch.equal(y, held)
    wc, ws = tokens.quantize_tokens(layer.weight.detach())
    assert torch.equal(y, tokens.linear_tokens(x.detach().to(dtype), wc, ws, layer.bias.detach()))
    y.backward(go)
    # the gradient of the weight in its own type: 16-bit values, sums in 32 bits that are not rounded to 16
    codes, scale = tokens.quantize_tokens(x.detach().to(dtype))
    values = codes.double() * scale.double()[:, None]
    exact, size = go.double().t() @ values, go.double().abs().t() @ values.abs()
    grad = layer.weight.grad
    assert grad.dtype == torch.float32 and torch.equal(grad, tokens.linear_tokens_grad_weight(go, codes, scale, torch.float32))
    assert ((grad.double() - exact).abs() <= (HALF_STEP[dtype] * 1.01 + 2.0 ** -23 * (M + 2)) * size).all()
    assert layer.bias.grad.dtype == torch.float32 and x.grad.dtype == torch.float32
    assert ((layer.bias.grad.double() - go.double().sum(0)).abs() <= 2.0 ** -23 * (M + 2) * go.double().abs().sum(0)).all()


@pytest.mark.gpu
def test_a_frozen_layer_keeps_nothing_of_its_input():
    layer = layers.QInt8Linear(1024, 64).to(DEV).bfloat16()
    x = torch.randn(4096, 1024, device=DEV).bfloat16().requires_grad_()
    layer(x)
    trained, kept = allocated(lambda: layer(x))
    assert kept >= 4096 * 1024                                              # (the codes)
    layer.weight.requires_grad_(False)
    y, kept = allocated(lambda: layer(x))
    assert kept <= y.numel() * 2 + 65536 and torch.equal(y, trained)
    go = torch.randn_like(y)
    y.backward(go)
    want = go.double() @ layer.weight.double()
    size = go.double().abs() @ layer.weight.double().abs()
    assert ((x.grad.double() - want).abs() <= 2.0 ** -23 * 66 * size + 2.0 ** -8 * want.abs() * 1.01).all()
    assert layer.weight.grad is None and layer.bias.grad is not None
    # and where only the weight is trained the gradient of the input is not made
    layer.weight.requires_grad_(True)
    layer(x.detach()).backward(go)
    assert layer.weight.grad is not None


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 70])
def test_a_frozen_layer_multiplies_the_weight_it_holds(M, monkeypatch):
    torch.manual_seed(2)
    layer = layers.QInt8Linear(64, 24).to(DEV)
    layer.weight.requires_grad_(False)
    x = torch.randn(M, 64, device=DEV, requires_grad=True)
    want = layer(x).detach()
    layer.hold_weight()
    rounded = []
    monkeypatch.setattr(tokens, "quantize_tokens", lambda t: rounded.append(t) or 1 / 0)
    y = layer(x)
    y.sum().backward()
    assert not rounded and torch.equal(y.detach(), want) and layer._held is not None
    monkeypatch.undo()
    with torch.inference_mode():
        layer.hold_weight()
    x.grad = None
    layer(x).sum().backward()
    assert x.grad is not None and layer._held is not None
    with torch.no_grad():
        layer.weight.mul_(2.0)
    assert torch.equal(layer(x).detach(), tokens.linear_tokens(x.detach(), *tokens.quantize_tokens(layer.weight), layer.bias.detach()))


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", [torch.optim.SGD, torch.optim.AdamW])
def test_a_hold_ends_when_the_weight_is_trained(optimizer):
    # (a fused optimizer's steps are not counted as changes of the tensor)
    torch.manual_seed(3)
    layer = layers.QInt8Linear(64, 24).to(DEV).eval()
    step = optimizer(layer.parameters(), lr=0.1, fused=True)
    x = torch.randn(5, 64, device=DEV)
    with torch.no_grad():
        before = layer.hold_weight()(x)
    layer(x).square().sum().backward()
    step.step()
    with torch.no_grad():
        got = layer(x)
        assert not torch.equal(got, before)
        assert torch.equal(got, tokens.linear_tokens(x, *tokens.quantize_tokens(layer.weight), layer.bias))


def test_a_hold_ends_when_weights_are_loaded():
    # whatever way load_state_dict takes to put them in place
    for swap in (False, True):
        torch.__future__.set_swap_module_params_on_conversion(swap)
        try:
            layer = layers.QInt8Linear(16, 4)
            layer._held = (layer.weight, layer.weight._version, None, None)
            layer.load_state_dict({k: torch.zeros_like(v) for k, v in layer.state_dict().items()})
            assert layer._held is None
        finally:
            torch.__future__.set_swap_module_params_on_conversion(False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_held_16_bit_layer_converts_its_bias_once(dtype, monkeypatch):
    torch.manual_seed(4)
    layer = layers.QInt8Linear(64, 24).to(DEV).to(dtype).eval()
    x = torch.randn(1, 64, device=DEV).to(dtype)
    given = []
    real = tokens.linear_tokens
    monkeypatch.setattr(tokens, "linear_tokens", lambda *a, **k: given.append(a[3]) or real(*a, **k))
    with torch.no_grad():
        want = layer(x)
        layer.hold_weight()
        assert torch.equal(layer(x), want) and torch.equal(layer(x), want)
        assert given[-1].dtype == torch.float32 and given[-1] is given[-2]
        layer.bias.add_(1.0)                                                # noticed
        after = layer(x)
        assert torch.equal(after, real(x, *tokens.quantize_tokens(layer.weight), layer.bias)) and not torch.equal(after, want)
        layer.hold_weight()
        layer.bias = nn.Parameter(torch.zeros_like(layer.bias))
        assert torch.equal(layer(x), real(x, *tokens.quantize_tokens(layer.weight), None))
        layer.hold_weight()
        layer.bias = None
        assert torch.equal(layer(x), real(x, *tokens.quantize_tokens(layer.weight), None))
    # a bias that is trained beside a frozen weight leaves the weight's hold alone
    layer = layers.QInt8Linear(64, 24).to(DEV).to(dtype)
    layer.weight.requires_grad_(False)
    step = torch.optim.SGD([layer.bias], lr=1.0, fused=True)
    layer.hold_weight()
    layer(x).sum().backward()
    step.step()
    with torch.no_grad():
        got = layer(x)
        assert torch.equal(got, real(x, *tokens.quantize_tokens(layer.weight), layer.bias)) and layer._held is not None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_without_compression_the_input_itself_is_kept(dtype):
    torch.manual_seed(5)
    config.compress_activation = False
    layer = layers.QInt8Linear(256, 48).to(DEV).to(dtype)
    x = torch.randn(20, 60, 256, device=DEV).to(dtype)
    go = torch.randn(20, 60, 48, device=DEV).to(dtype)
    layer(x)
    y, kept = allocated(lambda: layer(x))
    assert kept <= y.numel() * y.element_size() + 65536                     # nothing but the input that is there already
    assert torch.equal(y.detach(), tokens.linear_tokens(x, *tokens.quantize_tokens(layer.weight.detach()), layer.bias.detach()))
    y.backward(go)
    g, rows = go.double().reshape(-1, 48), x.double().reshape(-1, 256)
    exact, size = g.t() @ rows, g.abs().t() @ rows.abs()
    # exact products, 1200 additions in 32 bits, one rounding
    bound = 2.0 ** -23 * 1202 * size + HALF_STEP[dtype] * exact.abs() * 1.01 + 2.0 ** -25
    assert ((layer.weight.grad.double() - exact).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_batch_of_gradients_at_once(dtype):
    torch.manual_seed(6)
    layer = layers.QInt8Linear(64, 24).to(DEV).to(dtype)
    x = torch.randn(40, 64, device=DEV).to(dtype).requires_grad_()
    grads = torch.randn(3, 40, 24, device=DEV).to(dtype)
    wanted = (x, layer.weight, layer.bias)
    got = torch.autograd.grad(layer(x), wanted, grads, is_grads_batched=True)
    codes, scale = tokens.quantize_tokens(x.detach())
    values = (codes.float() * scale[:, None]).to(dtype).double()
    for i in range(3):
        g = grads[i].double()
        w = layer.weight.detach().double()
        for a, exact, size in ((got[0][i], g @ w, g.abs() @ w.abs()), (got[1][i], g.t() @ values, g.abs().t() @ values.abs()),
                               (got[2][i], g.sum(0), g.abs().sum(0))):
            assert a.dtype == dtype
            # sums of at most 40 terms in 32 bits, one rounding; fp16's kept values may be rounded by way of 32 bits
            assert ((a.double() - exact).abs() <= (2.0 ** -23 * 42 + 2.0 ** -23) * size + HALF_STEP[dtype] * exact.abs() * 1.01 + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradients_of_the_kernels_repeat_bit_for_bit(dtype):
    torch.manual_seed(7)
    linear, norm = layers.QInt8Linear(96, 200).to(DEV).to(dtype), layers.QGroupNorm(6, 96).to(DEV)
    rows, go = torch.randn(3000, 96, device=DEV).to(dtype), torch.randn(3000, 200, device=DEV).to(dtype)
    image, gi = (torch.randn(5, 30, 31, 96, device=DEV).to(dtype).permute(0, 3, 1, 2) for _ in range(2))
    first = None
    for _ in range(3):
        image = image.detach().requires_grad_()
        linear.zero_grad()
        norm.zero_grad()
        linear(rows).backward(go)
        norm(image, silu=True).backward(gi)
        got = [image.grad, norm.weight.grad, norm.bias.grad] + ([linear.weight.grad] if dtype != torch.float32 else [])
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_to_channels_last_of_every_number_of_dimensions():
    for shape in ((2, 3), (2, 3, 5), (2, 3, 5, 4), (2, 3, 2, 3, 4)):
        x = torch.randn(shape)
        y = to_channels_last(x)
        assert torch.equal(x, y) and y.movedim(1, -1).is_contiguous() and to_channels_last(y) is y
    x = torch.randn(3, 2).t()
    y = to_channels_last(x)
    assert torch.equal(x, y) and y.is_contiguous()
