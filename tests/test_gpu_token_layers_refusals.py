"""Inputs that the plain layers refuse, under the layers that stand in for them."""
import pytest
import torch

from actnn_amd import layers


def test_a_single_value_is_refused_as_by_the_plain_layer():
    # (before anything is asked of the GPU)
    for shape, groups in (((1, 4), 4), ((1, 6, 1, 1), 6)):
        for layer in (torch.nn.GroupNorm(groups, shape[1]), layers.QGroupNorm(groups, shape[1])):
            with pytest.raises(ValueError, match="more than 1 value"):
                layer(torch.zeros(shape))
