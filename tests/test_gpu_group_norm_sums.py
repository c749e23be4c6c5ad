"""The group norm's sums over planes so large that a thread adds up thousands of pixels."""
import pytest
import torch

from actnn_amd.cpp_extension import backward_func as bf

DEV = "cuda:0"
# Additions in a row that a sum is made of: 128, one for every 128 pixels of a thread (at most 33 here), 8 rows of threads, 64 slices
# by as many lanes: below 256, each rounding to 2^-24 of what has been summed.
SUMMED = 2.0 ** -16


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((1, 128, 1448, 1448), torch.float32), ((1, 1024, 512, 511), torch.float32),
                                          ((1, 256, 1448, 1448), torch.bfloat16)])
def test_sums_of_thousands_of_equal_pixels(shape, dtype):
    # equal terms: every addition in a row rounds the same way, nothing cancels (one group: as few threads as there can be)
    N, C, H, W = shape
    print(f"[group_norm] {shape} {dtype}", flush=True)
    x = torch.zeros(N, H, W, C, dtype=dtype, device=DEV).permute(0, 3, 1, 2)
    b = torch.linspace(-1.5, 1.5, C, device=DEV)
    w = torch.linspace(0.5, 1.5, C, device=DEV)
    dy = torch.linspace(0.7, 1.3, C, device=DEV).to(dtype).view(1, 1, 1, C).expand(N, H, W, C).contiguous().permute(0, 3, 1, 2)
    mean, rstd = torch.full((N, 1), -0.73, device=DEV), torch.full((N, 1), 0.61, device=DEV)
    dx, dw, db = bf.hip_group_norm_backward(dy, None, None, 1, w, b, mean, rstd, "silu", input=x)
    n = float(torch.tensor(0.73)) * float(torch.tensor(0.61))
    z = n * w.double() + b.double()
    s = torch.sigmoid(z)
    dz = dy[0, :, 0, 0].double() * s * (1 + z * (1 - s))
    P = N * H * W
    # a term: the slope of order one by an approximate sigmoid, 2^-20 of |dy|
    off = 2.0 ** -20 * dy[0, :, 0, 0].double().abs() * P
    assert ((db.double() - dz * P).abs() <= SUMMED * dz.abs() * P + off).all(), float(((db.double() - dz * P).abs() / (dz.abs() * P)).max())
    assert ((dw.double() - dz * n * P).abs() <= n * (SUMMED * dz.abs() * P + off)).all()
    u, r = dz * w.double(), float(torch.tensor(0.61))
    ex = r * (u - (1 + n * n) * u.mean())
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    assert ((dx[0, :, 5, 7].double() - ex).abs() <= half * ex.abs() + r * (SUMMED + 2.0 ** -20) * 2 * 2).all()
