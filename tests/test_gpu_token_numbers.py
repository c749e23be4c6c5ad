"""8-bit tokens at the ends of the types' ranges, and the same values wherever codes are turned back into them."""
import numpy as np
import pytest
import torch

from actnn_amd.cpp_extension import tokens

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K", [256, 1003])
def test_what_is_read_back_is_what_the_weight_gradient_multiplies(K, dtype):
    torch.manual_seed(K)
    M = 3000
    x = torch.randn(M, K, device=DEV) * torch.randn(M, 1, device=DEV).mul_(1.5).exp_()
    x[:, 0] = x.abs().amax(1)
    codes, scale = tokens.quantize_tokens(x)
    # every code with every scale
    codes[:, 1:] = (torch.arange(K - 1, device=DEV) % 255 - 127).to(torch.int8)
    back = tokens.dequantize_tokens(codes, scale, dtype)
    exact = codes.cpu().double() * scale.cpu().double()[:, None]
    if dtype == torch.float16:                                                             # one rounding (numpy's)
        assert torch.equal(back.cpu(), torch.from_numpy(exact.numpy().astype(np.float16)))
    else:                                                                                  # by way of 32 bits
        assert torch.equal(back.cpu(), exact.float().bfloat16())
    one = torch.zeros(M, 8, dtype=dtype, device=DEV)
    # eight tokens at a time, each with an output of its own
    for m in range(0, M, 8):
        one.zero_()
        one[m:m + 8] = torch.eye(8, device=DEV)
        assert torch.equal(tokens.linear_tokens_grad_weight(one, codes, scale), back[m:m + 8]), m


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,O", [(1, 4096, 64), (3, 1003, 40), (20, 4096, 33), (70, 8192, 64), (300, 2048, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_tokens_with_small_weights_and_the_other_way_round(M, K, O, dtype):
    # the sum times one scale passes the largest number, the result does not: y is of order 2^100
    for by, weight_by in ((2.0 ** 115, 2.0 ** -20), (2.0 ** -20, 2.0 ** 115), (2.0 ** 50, 2.0 ** 50)):
        x = torch.full((M, K), by, device=DEV).to(dtype)
        x[:, 1] = -by / 2
        codes, scale = tokens.quantize_tokens(x)
        wcodes, wscale = tokens.quantize_tokens(torch.full((O, K), weight_by, device=DEV) * torch.linspace(0.5, 1, O, device=DEV)[:, None])
        exact = (codes.double() @ wcodes.double().t()) * scale.double()[:, None] * wscale.double()
        assert exact.abs().max() < 3e38 and exact.abs().max() > 1e27
        for y in (tokens.linear_tokens(x, wcodes, wscale), tokens.matmul_tokens(codes, scale, wcodes, wscale, None, dtype)):
            half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
            assert ((y.double() - exact).abs() <= (3.01 * 2.0 ** -24 + half * 1.01) * exact.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [4, 20, 300])
def test_a_large_token_leaves_its_neighbours_as_they_are(M):
    torch.manual_seed(M)
    x = torch.randn(M, 512, device=DEV)
    wcodes, wscale = tokens.quantize_tokens(torch.randn(300, 512, device=DEV) * 2.0 ** -30)
    alone = tokens.linear_tokens(x, wcodes, wscale)
    x[M // 2] *= 2.0 ** 120
    y = tokens.linear_tokens(x, wcodes, wscale)
    rest = [m for m in range(M) if m != M // 2]
    assert torch.equal(y[rest], alone[rest])
    # the same converted sum times the same two numbers, in either order: two roundings to 2^-24 each, on both sides
    got, want = y[M // 2].double(), alone[M // 2].double() * 2.0 ** 120
    assert ((got - want).abs() <= 4.01 * 2.0 ** -24 * want.abs()).all()
