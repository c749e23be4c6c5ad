"""The same values wherever codes of 8-bit tokens are turned back into them."""
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
