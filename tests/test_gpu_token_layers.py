"""The 8-bit token layers and the group norm as a model uses them: alone, together, converted by QModule, captured."""
import copy
import io

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import actnn_amd as actnn
from actnn_amd import layers
from actnn_amd.conf import config
from actnn_amd.cpp_extension import tokens
from actnn_amd.utils import to_channels_last
from oracle import group_norm as oracle_gn

DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def fresh_config():
    config.reset()
    yield
    config.reset()


def linear_oracle(layer, x, go):
    """Output and gradients of QInt8Linear in 64 bits, from the layer's own codes (whose exactness has its own tests)."""
    codes, scale = tokens.quantize_tokens(x)
    wcodes, wscale = tokens.quantize_tokens(layer.weight.detach())
    xv, wv = codes.double() * scale.double()[..., None], wcodes.double() * wscale.double()[:, None]
    y = xv @ wv.t() + (0 if layer.bias is None else layer.bias.detach().double())
    g = go.double().reshape(-1, go.shape[-1])
    rows = xv.reshape(-1, xv.shape[-1])
    return (y, go.double() @ layer.weight.detach().double(), g.t() @ rows, g.sum(0),
            g.abs() @ layer.weight.detach().double().abs(), g.abs().t() @ rows.abs(), g.abs().sum(0), xv.abs() @ wv.abs().t())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,K,O,bias", [((70,), 100, 36, True), ((3, 5), 64, 17, True), ((2, 3, 100), 40, 64, False)])
def test_linear_layer(lead, K, O, bias, dtype):
    torch.manual_seed(1)
    layer = layers.QInt8Linear(K, O, bias).to(DEV).to(dtype)
    x = (2 * torch.randn(*lead, K, device=DEV)).to(dtype).requires_grad_()
    go = torch.randn(*lead, O, device=DEV).to(dtype)
    y = layer(x)
    y.backward(go)
    ey, ex, ew, eb, sx, sw, sb, sy = linear_oracle(layer, x.detach(), go)
    h, n = HALF_STEP[dtype], x.numel() // K
    assert y.dtype == dtype and ((y.double() - ey).abs() <= 8 * 2.0 ** -24 * sy + h * ey.abs() * 1.01 + 2.0 ** -24 * sy.max()).all()
    # products of the library: each term exact, sums in fp32, one rounding
    assert ((x.grad.double() - ex).abs() <= 2.0 ** -23 * (O + 2) * sx.view(ex.shape) + h * ex.abs() * 1.01 + 2.0 ** -25).all()
    # the kept values are rounded to the gradient's type (16-bit types) before they are multiplied
    kept = 0.0 if dtype == torch.float32 else h
    assert ((layer.weight.grad.double() - ew).abs() <= (kept + 2.0 ** -23 * (n + 2)) * sw + h * ew.abs() * 1.01 + 2.0 ** -25).all()
    if bias:
        assert ((layer.bias.grad.double() - eb).abs() <= 2.0 ** -23 * (n + 2) * sb + h * eb.abs() * 1.01 + 2.0 ** -25).all()


@pytest.mark.gpu
def test_linear_layer_gradients_against_differences():
    # in full precision with a weight that codes hold exactly, the output is linear in the input's kept values and in the weight
    torch.manual_seed(2)
    layer = layers.QInt8Linear(16, 8).to(DEV)
    x = torch.randint(-127, 128, (6, 16), device=DEV).float()
    x[:, 0] = 127.0
    with torch.no_grad():
        layer.weight.copy_(torch.randint(-127, 128, (8, 16), device=DEV).float() / 64)
        layer.weight[:, 1] = 127.0 / 64
    x.requires_grad_()
    go = torch.randn(6, 8, device=DEV)
    layer(x).backward(go)
    for m, k in ((0, 3), (5, 15)):
        step = torch.zeros_like(x)
        step[m, k] = 1.0 if x[m, k] < 126 else -1.0                    # from one code to its neighbour
        with torch.no_grad():
            numeric = ((layer(x + step) - layer(x)).double() * go.double()).sum() / step[m, k].double()
        # outputs up to 127 * 127 * 16 / 64 rounded to 24 bits, eight of them
        assert abs(float(numeric) - float(x.grad[m, k])) <= 8 * 2 * 2.0 ** -23 * 127 * 127 / 4 * float(go.abs().max())
    for o, k in ((0, 2), (7, 9)):
        step = torch.zeros_like(layer.weight)
        step[o, k] = (1.0 if layer.weight[o, k] < 126 / 64 else -1.0) / 64
        with torch.no_grad():
            before = layer(x)
            layer.weight += step
            numeric = ((layer(x) - before).double() * go.double()).sum() / step[o, k].double()
            layer.weight -= step
        assert abs(float(numeric) - float(layer.weight.grad[o, k])) <= 64 * 6 * 2 * 2.0 ** -23 * 127 * 127 / 4 * float(go.abs().max())


@pytest.mark.gpu
def test_linear_layer_keeps_a_byte_a_value():
    layer = layers.QInt8Linear(1024, 64).to(DEV).bfloat16()
    x = torch.randn(4096, 1024, device=DEV).bfloat16().requires_grad_()
    layer(x)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = layer(x)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert 4096 * 1024 <= kept <= 4096 * 1024 + 4096 * 4 + 65536


@pytest.mark.gpu
def test_held_weights():
    torch.manual_seed(3)
    layer = layers.QInt8Linear(96, 40).to(DEV).bfloat16().eval()
    x = torch.randn(2, 96, device=DEV).bfloat16()
    with torch.no_grad():
        want = layer(x)
        layer.hold_weight()
        assert layer._held is not None and torch.equal(layer(x), want)
        layer.weight.mul_(2.0)                                          # noticed: rounded anew
        assert torch.equal(layer(x), layers.ext_tokens.linear_tokens(
            x, *tokens.quantize_tokens(layer.weight), layer.bias)) and layer._held is None
        layer.hold_weight()
        layer.load_state_dict({"weight": torch.ones_like(layer.weight), "bias": torch.zeros_like(layer.bias)})
        assert torch.equal(layer(x), layers.ext_tokens.linear_tokens(x, *tokens.quantize_tokens(torch.ones_like(layer.weight)), None))
        layer.hold_weight()
        layer.weight = nn.Parameter(torch.zeros_like(layer.weight))
        assert (layer(x) == 0).all()
        layer.hold_weight()
        twin = copy.deepcopy(layer)
        assert twin._held is None and layer._held is not None
        buffer = io.BytesIO()
        torch.save(layer.state_dict(), buffer)
        layer.float()
        assert layer._held is None
        layer.hold_weight().train()
        assert layer._held is None


@pytest.mark.gpu
def test_weights_held_in_inference_mode():
    with torch.inference_mode():
        layer = layers.QInt8Linear(64, 8).to(DEV)
        x = torch.randn(3, 64, device=DEV)
        want = layer(x)
        assert torch.equal(layer.hold_weight()(x), want) and layer._held is not None


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    layer, norm = layers.QInt8Linear(16, 8).to(DEV), layers.QGroupNorm(2, 16).to(DEV)
    x = torch.randn(4, 16, device=DEV, requires_grad=True)
    for f in (lambda: layer(x), lambda: norm(x)):
        (g,) = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("compress", [True, False])
@pytest.mark.parametrize("shape,groups", [((3, 24, 10, 6), 4), ((2, 33, 7), 11), ((5, 16), 2), ((2, 8, 3, 4, 5), 2)])
def test_group_norm_layer(shape, groups, compress, dtype):
    torch.manual_seed(4)
    config.compress_activation = compress
    gn = layers.QGroupNorm(groups, shape[1]).to(DEV)
    with torch.no_grad():
        gn.weight.normal_(1.0, 0.2)
        gn.bias.normal_(0.0, 0.2)
    x0 = torch.randn(shape, device=DEV).to(dtype)
    go = torch.randn(shape, device=DEV).to(dtype)
    for layout in (x0, to_channels_last(x0)):
        x = layout.detach().clone(memory_format=torch.preserve_format).requires_grad_()
        gn.zero_grad()
        y = layers.gn_silu(gn, nn.SiLU(), x)
        y.backward(go)
        ey, mean, rstd = oracle_gn.forward(x.detach(), groups, gn.weight.detach(), gn.bias.detach(), gn.eps, "silu")
        values = x.detach()
        if compress:
            q, s = oracle_gn.kept(values, groups)
            values = (q * s[:, :, None].expand(shape[0], groups, shape[1] // groups).reshape(shape[:2] + (1,) * (len(shape) - 2))).to(DEV)
        ex, ew, eb = oracle_gn.backward(go, values, mean, rstd, groups, gn.weight.detach(), gn.bias.detach(), "silu")
        h = HALF_STEP[dtype]
        # values of order one, statistics of hundreds of values: 2^-16 holds all sums (each of fewer than 256 additions)
        for got, exact in ((y, ey), (x.grad, ex), (gn.weight.grad, ew), (gn.bias.grad, eb)):
            half = h if got.dtype == dtype else 2.0 ** -24
            assert ((got.double() - exact).abs() <= half * exact.abs() + 2.0 ** -16 * (1 + exact.abs().max()) + 2.0 ** -25).all()
        with torch.no_grad():
            assert torch.equal(gn(x, silu=True), y)
            # the two calls round once more in between
            apart = F.silu(gn(x))
            assert ((apart.double() - ey).abs() <= 3 * h * (1 + ey.abs()) + 2.0 ** -16 * (1 + ey.abs().max())).all()
    plain = nn.GroupNorm(groups, shape[1]).to(DEV)
    assert torch.equal(layers.gn_silu(plain, nn.SiLU(), x0.float()), F.silu(plain(x0.float())))


class Block(nn.Module):
    """Group norm + SiLU over pixels, then a two-layer perceptron over the channels of each pixel, added to its input."""

    def __init__(self, channels=48, groups=6, hidden=96):
        super().__init__()
        self.norm, self.act = nn.GroupNorm(groups, channels), nn.SiLU()
        self.up, self.down = nn.Linear(channels, hidden), nn.Linear(hidden, channels)

    def forward(self, x):
        h = layers.gn_silu(self.norm, self.act, x).permute(0, 2, 3, 1)
        return x + self.down(F.silu(self.up(h))).permute(0, 3, 1, 2)


def convert():
    config.enable_int8_linear = config.enable_quantized_gn = True
    torch.manual_seed(5)
    return actnn.QModule(nn.Sequential(Block(), Block()), channels_last=True).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [None, torch.bfloat16, torch.float16])
def test_layers_together_in_a_converted_model(autocast):
    model = convert()
    assert [type(m) for m in model.modules() if isinstance(m, (nn.GroupNorm, nn.Linear))] == [layers.QGroupNorm, layers.QInt8Linear, layers.QInt8Linear] * 2
    plain = nn.Sequential(Block(), Block()).to(DEV)
    plain.load_state_dict(model.state_dict())
    x = torch.randn(2, 48, 12, 10, device=DEV)
    go = torch.randn_like(x)
    grads = []
    for m in (model, plain):
        m.zero_grad()
        xi = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=autocast or torch.bfloat16, enabled=autocast is not None):
            y = m(xi)
        y.float().backward(go)
        grads.append([y.detach().float(), xi.grad] + [p.grad for p in m.parameters()])
    # 8 bits a factor: a rounding of a 254th of a row's largest value, about 3 of its standard deviations, is 0.7 % of the
    # values' size in the 2-norm; two such factors, two products a block and two blocks, and the slope of what follows: below 6 %
    for got, want in zip(*grads):
        assert torch.isfinite(got).all() and got.shape == want.shape
        assert (got - want).norm() <= 0.06 * want.norm()
    # and a step is the same step each time
    first = [g.clone() for g in grads[0]]
    model.zero_grad()
    xi = x.clone().requires_grad_()
    with torch.autocast("cuda", dtype=autocast or torch.bfloat16, enabled=autocast is not None):
        y = model(xi)
    y.float().backward(go)
    again = [y.detach().float(), xi.grad] + [p.grad for p in model.parameters()]
    for a, b in zip(first[:1], again[:1]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_training_step_captured():
    model = convert().bfloat16()
    x = torch.randn(2, 48, 8, 8, device=DEV).bfloat16().contiguous(memory_format=torch.channels_last)
    params = list(model.parameters())

    def step():
        return torch.autograd.grad(model(x).float().square().sum(), params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in grads]
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            # (the library may choose another product inside a capture: fp32 sums in another order, one rounding)
            assert (a.float() - b.float()).norm() <= 2.0 ** -7 * b.float().norm() + 1e-6, i


@pytest.mark.gpu
def test_conversion_is_off_unless_asked():
    model = actnn.QModule(nn.Sequential(Block())).to(DEV)
    kinds = [type(m) for m in model.modules() if isinstance(m, (nn.GroupNorm, nn.Linear))]
    assert kinds == [nn.GroupNorm, layers.QLinear, layers.QLinear]


def test_to_channels_last_and_conversion_on_the_cpu():
    for shape in ((2, 3), (2, 3, 5), (2, 3, 5, 4), (2, 3, 2, 3, 4)):
        x = torch.randn(shape)
        y = to_channels_last(x)
        assert torch.equal(x, y) and y.movedim(1, -1).is_contiguous() and to_channels_last(y) is y or len(shape) == 2
    config.enable_int8_linear = config.enable_quantized_gn = True
    model = actnn.QModule(nn.Sequential(Block()))
    assert isinstance(model.model[0].norm, layers.QGroupNorm) and isinstance(model.model[0].up, layers.QInt8Linear)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        model(torch.zeros(1, 48, 2, 2))
