"""The weight gradient from 8-bit tokens against the same sum in 64 bits over the values the kernel multiplies: the codes'
values rounded to the gradient's type, so that what is left is the fp32 sum and the output's rounding."""
import numpy as np
import pytest
import torch

from actnn_amd.cpp_extension import tokens

DEV = "cuda:0"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(M, O, I, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, I, generator=gen, device=DEV) * torch.randn(M, 1, generator=gen, device=DEV).exp()
    if M > 3:
        x[1] = 0
    g = (torch.randn(M, O, generator=gen, device=DEV) * 0.1).to(dtype)
    return (g, *tokens.quantize_tokens(x))


def kept_values(codes, scale, dtype):
    """What the kernel multiplies: fp16 rounded once (numpy's conversion), bf16 by way of 32 bits."""
    if dtype == torch.float16:
        exact = codes.double() * scale.double()[..., None]
        return torch.from_numpy(exact.cpu().numpy().astype(np.float16)).to(codes.device).double()
    return (codes.float() * scale[..., None]).to(dtype).double()


def check(gw, g, codes, scale, out):
    values = kept_values(codes, scale, g.dtype).reshape(-1, codes.shape[-1])
    gd = g.double().reshape(-1, g.shape[-1])
    exact = gd.t() @ values
    size = gd.abs().t() @ values.abs()
    M = gd.shape[0]
    # every one of the M - 1 additions and products rounds (or truncates: a step, not half of one) what has been summed so far
    bound = 2.0 ** -23 * (M + 2) * size + HALF_STEP[out] * exact.abs() * 1.01 + (2.0 ** -25 if out == torch.float16 else 0.0)
    assert gw.dtype == out and gw.shape == exact.shape
    err = (gw.double() - exact).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())
    if out == torch.float32 and M >= 64:
        # rounding errors do not all point one way: the 2-norm is far inside
        assert err.norm() <= 2.0 ** -23 * (M ** 0.5 + 2) * size.norm()


SHAPES = [(1, 8, 16), (1, 1, 1), (2, 3, 5), (3, 7, 33), (63, 64, 128), (64, 128, 128), (65, 129, 130), (100, 100, 784), (1000, 100, 784),
          (257, 1, 300), (300, 260, 1), (513, 250, 257), (2048, 40, 40), (130, 1000, 515), (512, 512, 512), (1030, 512, 768), (4096, 256, 256), (640, 2048, 1100),
          (2048, 2048, 2048), (2177, 2056, 2100), (4100, 2051, 2033), (5000, 1800, 2300)]        # the large tiles, with and without splits


@pytest.mark.gpu
@pytest.mark.parametrize("M,O,I", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradient(M, O, I, dtype):
    g, codes, scale = make(M, O, I, dtype, M + O + I)
    for out in (dtype, torch.float32):
        print(f"[tokens_grad] {M}x{O}x{I} {dtype} -> {out}", flush=True)
        gw = tokens.linear_tokens_grad_weight(g, codes, scale, out)
        check(gw, g, codes, scale, out)
        assert torch.equal(gw, tokens.linear_tokens_grad_weight(g, codes, scale, out))      # no order that changes


@pytest.mark.gpu
def test_gradient_is_the_formulas_difference():
    # sum_o,m g y is linear in the weight: its difference quotient is the gradient up to the sums' rounding
    M, O, I = 40, 6, 20
    g, codes, scale = make(M, O, I, torch.float16, 3)
    gw = tokens.linear_tokens_grad_weight(g, codes, scale, torch.float32).double()
    values = kept_values(codes, scale, torch.float16)
    w = torch.randn(O, I, device=DEV, dtype=torch.float64)
    loss = lambda w: (g.double() * (values @ w.t())).sum()  # noqa: E731
    for o, i in ((0, 0), (3, 7), (5, 19)):
        step = torch.zeros_like(w)
        step[o, i] = 0.5
        numeric = (loss(w + step) - loss(w - step)).item()
        assert abs(numeric - gw[o, i].item()) <= 2.0 ** -23 * (M + 2) * (g[:, o].double().abs() @ values[:, i].abs()).item() + 1e-9


# splits of any number; gradients whose rows are no whole chunks, copied and as they are
@pytest.mark.gpu
@pytest.mark.parametrize("M,O,I", [(1500, 327, 3200), (1156, 673, 1728), (900, 1001, 3000), (4000, 1001, 1024), (5000, 60, 500), (3000, 515, 700)])
def test_gradient_between_the_kernels(M, O, I):
    test_gradient(M, O, I, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [70, 700])
def test_layouts_strides_and_leading_dimensions(M, dtype):
    g, codes, scale = make(M, 96, 80, dtype, 9)
    want = tokens.linear_tokens_grad_weight(g, codes, scale)
    wide = torch.full((M, 200), float("nan"), dtype=dtype, device=DEV)
    for at in (1, 7, 8, 104):
        wide[:, at:at + 96] = g
        assert torch.equal(tokens.linear_tokens_grad_weight(wide[:, at:at + 96], codes, scale), want)
    assert torch.equal(tokens.linear_tokens_grad_weight(g.t().contiguous().t(), codes, scale), want)
    assert torch.equal(tokens.linear_tokens_grad_weight(g, codes.t().contiguous().t(), scale), want)
    lead = tokens.linear_tokens_grad_weight(g.view(10, -1, 96), codes.unflatten(0, (10, -1)), scale.view(10, -1))
    assert torch.equal(lead, want)
    even = tokens.linear_tokens_grad_weight(g[:1].expand(M, 96), codes, scale)
    assert torch.equal(even, tokens.linear_tokens_grad_weight(g[:1].expand(M, 96).contiguous(), codes, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 65, 257, 1023, 2175])
@pytest.mark.parametrize("O,I", [(16, 48), (264, 512), (2000, 2048)])
def test_infinite_gradients_stay_where_they_are(M, O, I):
    # an infinite gradient of the last token spoils its own output alone, and as an infinity
    g, codes, scale = make(M, O, I, torch.bfloat16, 4)
    codes[M - 1] = 3
    want = tokens.linear_tokens_grad_weight(g, codes, scale)
    g[M - 1, 5] = float("inf")
    gw = tokens.linear_tokens_grad_weight(g, codes, scale)
    assert torch.isposinf(gw[5]).all()
    rest = [o for o in range(O) if o != 5]
    assert torch.equal(gw[rest], want[rest])


@pytest.mark.gpu
def test_no_tokens_and_no_outputs():
    codes, scale = tokens.quantize_tokens(torch.zeros(0, 24, device=DEV))
    gw = tokens.linear_tokens_grad_weight(torch.zeros(0, 5, device=DEV, dtype=torch.float16), codes, scale)
    assert gw.shape == (5, 24) and (gw == 0).all()
    codes, scale = tokens.quantize_tokens(torch.zeros(4, 24, device=DEV))
    assert tokens.linear_tokens_grad_weight(torch.zeros(4, 0, device=DEV, dtype=torch.float16), codes, scale).shape == (0, 24)


@pytest.mark.gpu
@pytest.mark.parametrize("M,O,I", [(512, 64, 200), (700, 520, 512), (2100, 2000, 2003)])
def test_captured_and_replayed(M, O, I):
    g, codes, scale = make(M, O, I, torch.bfloat16, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tokens.linear_tokens_grad_weight(g, codes, scale)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gw = tokens.linear_tokens_grad_weight(g, codes, scale)
    for i in range(4):
        g.copy_(torch.randn(M, O, device=DEV))
        scale.mul_(1.25)
        graph.replay()
        want = tokens.linear_tokens_grad_weight(g, codes, scale)
        torch.cuda.synchronize()
        assert torch.equal(gw, want), i


def test_refusals_on_the_cpu():
    c, s = torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        tokens.linear_tokens_grad_weight(torch.zeros(4, 8, dtype=torch.float16), c, s)


@pytest.mark.gpu
def test_refusals():
    c, s = torch.zeros(4, 16, dtype=torch.int8, device=DEV), torch.zeros(4, device=DEV)
    g = torch.zeros(4, 8, device=DEV, dtype=torch.bfloat16)
    for args, text in (((g.float(), c, s), "type of grad_output"), ((g[:3], c, s), "same tokens"), ((g.view(2, 2, 8), c, s), "same tokens"),
                       ((g, c.float(), s), "type of codes"), ((g, c, s[:2]), "one value for each row"), ((g, c.cpu(), s), "CUDA"),
                       ((g, c, s, torch.float16), "in the type of grad_output"), ((g, c, s, torch.float64), "float32, float16 or bfloat16")):
        with pytest.raises(RuntimeError, match=text):
            tokens.linear_tokens_grad_weight(*args)


def test_c_abi_refuses_bad_sizes(lib):
    f = lib.actnn_tokens_grad_weight
    assert f(None, 8, None, 16, None, None, 4, 0, 16, 1, 1, None, 0, None) == 0
    assert f(None, 8, None, 16, None, None, 4, 8, 16, 0, 0, None, 0, None) == -2          # fp32 gradients
    assert f(None, 8, None, 16, None, None, 4, 8, 16, 1, 2, None, 0, None) == -2          # another 16-bit result
    assert f(None, 8, None, 16, None, None, 4, 8, 17, 1, 1, None, 0, None) == -1          # rows shorter than I
    assert f(None, 8, None, 24, None, None, 4, 8, 16, 1, 1, None, 0, None) == -1          # no multiple of 16
    assert f(None, 8, None, 16, None, None, 4, 8, 16, 1, 1, None, 0, None) == -1          # null pointers
    assert f(16, 8, 16, 16, 16, 16, 1, 0x7fffff00, 16, 1, 1, None, 0, None) == -1         # more blocks than a launch takes
    assert f(16, 8, 16, 16, 16, 16, 0, 8, 16, 1, 1, None, 0, None) == -1                  # no tokens
    assert f(16, 1, 16, 16, 16, 16, 2, 1, 16, 1, 1, None, 0, None) == -1                  # below 16 bytes without room
    assert f(16, 8, 8, 16, 16, 16, 4, 8, 16, 1, 1, None, 0, None) == -4
    assert lib.actnn_tokens_grad_weight_workspace_bytes(1000, 100, 784) > 0
