"""64-bit restatement of the 8-bit token operators (CPU, numpy / torch float64)."""
import torch


def codes(x, dims=(-1,)):
    """(codes float64, scale float64 without `dims` kept) of x over `dims`: sign(x) floor(127 |x| / top + 1/2)."""
    v = x.detach().cpu().double()
    top = v.abs().amax(dim=dims, keepdim=True)
    bad = ~torch.isfinite(v).all(dim=dims[0], keepdim=True) if len(dims) == 1 else ~torch.isfinite(v.sum(dim=dims, keepdim=True))
    dead = top < 2.0 ** -100
    safe = torch.where(bad | dead, torch.ones_like(top), top)
    # 254 |x| / top, its whole part decides: exact in float64 (the products are, and a quotient that is no whole number is
    # at least 2^-33 of itself away from one)
    doubled = torch.floor(254.0 * v.abs() / safe)
    q = torch.floor((doubled + 1.0) / 2.0) * torch.sign(v)
    q = torch.where(bad | dead, torch.zeros_like(q), q)
    scale = torch.where(bad, torch.full_like(top, float("nan")), torch.where(dead, torch.zeros_like(top), top / 127.0))
    return q, scale
