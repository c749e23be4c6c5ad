"""Inputs that the plain layers refuse, under the layers that stand in for them."""
import pytest
import torch

from actnn_amd import layers
from actnn_amd.cpp_extension import backward_func as bf
from actnn_amd.cpp_extension import tokens


def test_a_single_value_is_refused_as_by_the_plain_layer():
    # (before anything is asked of the GPU)
    for shape, groups in (((1, 4), 4), ((1, 6, 1, 1), 6)):
        for layer in (torch.nn.GroupNorm(groups, shape[1]), layers.QGroupNorm(groups, shape[1])):
            with pytest.raises(ValueError, match="more than 1 value"):
                layer(torch.zeros(shape))


def test_tensors_without_memory_are_refused():
    # (a view of one has an address that is not zero: nothing may be launched with it; refused before anything is asked of the GPU)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(4, 32, device="cuda")[1:]
        c, s = torch.empty(4, 32, dtype=torch.int8, device="cuda")[1:], torch.empty(4, device="cuda")[1:]
        m = torch.empty(4, 2, device="cuda")[1:]
    for call in (lambda: tokens.quantize_tokens(x), lambda: tokens.dequantize_tokens(c, s), lambda: tokens.matmul_tokens(c, s, c, s),
                 lambda: tokens.linear_tokens(x, c, s), lambda: tokens.linear_tokens_grad_weight(x.half(), c, s),
                 lambda: bf.hip_group_norm_forward(x, 2, None, None, 1e-5),
                 lambda: bf.hip_group_norm_backward(x, None, None, 2, None, None, m, m, input=x)):
        with pytest.raises(RuntimeError, match="has no memory to read"):
            call()
