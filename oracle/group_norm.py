"""64-bit restatement of the group norm with its activation and of its backward pass (CPU or GPU, torch float64)."""
import torch

from . import tokens


def forward(x, groups, weight, bias, eps, activation):
    """-> (y, mean [N, G], rstd [N, G]) in float64."""
    N, C = x.shape[:2]
    v = x.double().reshape(N, groups, -1)
    mean = v.mean(2, keepdim=True)
    rstd = ((v - mean).square().mean(2, keepdim=True) + eps).rsqrt()
    shape = (1, C) + (1,) * (x.dim() - 2)
    z = ((v - mean) * rstd).view(x.shape)
    if weight is not None:
        z = z * weight.double().view(shape)
    if bias is not None:
        z = z + bias.double().view(shape)
    return (z * torch.sigmoid(z) if activation == "silu" else z), mean[:, :, 0], rstd[:, :, 0]


def kept(x, groups):
    """The codes of x, one scale for each sample and group, and that scale [N, G]."""
    q, s = tokens.codes(x.reshape(x.shape[0], groups, -1))
    return q.view(x.shape), s[:, :, 0]


def backward(dy, values, mean, rstd, groups, weight, bias, activation):
    """-> (dx, dw, db) at the saved input `values`, with the forward pass's mean and rstd [N, G], in float64."""
    N, C = values.shape[:2]
    shape = (1, C) + (1,) * (values.dim() - 2)
    w = torch.ones(C, dtype=torch.float64, device=dy.device) if weight is None else weight.double()
    b = torch.zeros(C, dtype=torch.float64, device=dy.device) if bias is None else bias.double()
    n = ((values.double().reshape(N, groups, -1) - mean.double()[:, :, None]) * rstd.double()[:, :, None]).view(values.shape)
    dz = dy.double()
    if activation == "silu":
        z = n * w.view(shape) + b.view(shape)
        s = torch.sigmoid(z)
        dz = dz * (s * (1 + z * (1 - s)))
    dims = [0] + list(range(2, values.dim()))
    u = (dz * w.view(shape)).reshape(N, groups, -1)
    ng = n.reshape(N, groups, -1)
    dx = rstd.double()[:, :, None] * (u - u.mean(2, keepdim=True) - ng * (u * ng).mean(2, keepdim=True))
    return dx.view(values.shape), (dz * n).sum(dims), dz.sum(dims)
