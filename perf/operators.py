"""The workloads that the 8-bit token operators and the group norm are measured on.

A token is a row of features: a word's hidden state, or the channels of one pixel in the channels-last layout.
Kinds:

  checkpoint   tokens written in 8 bits and read back: one scale for each token, codes -127 .. 127
  linear       a linear layer's product in 8-bit integers, from tokens in full precision and a weight whose codes
               and scales (one for each output channel) the program keeps
  linear_grad  the weight gradient from the output gradient and the tokens as the checkpoint holds them
  norm         group norm with its activation, channels last, forward alone
  norm_train   the same forward and backward, the input kept in 8 bits in between (one scale for each sample and group)

Rounding to codes: halves away from zero, of 127 times the value over the largest magnitude that shares its scale.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
SMALLEST = 2.0 ** -100      # magnitudes below count as zero where a scale is made
EPS = 1e-5


def listed():
    return [
        # the input of the repository's fully connected benchmark, as it is saved for the backward pass
        dict(name="checkpoint_bf16_large", kind="checkpoint", dtype="bf16", tokens=8192, features=4096),
        # a small batch of rows of odd length in full precision: calls of a few microseconds
        dict(name="checkpoint_f32_odd", kind="checkpoint", dtype="f32", tokens=333, features=1003),
        # one token of a program that generates: bound by reading the weight
        dict(name="linear_bf16_one_token", kind="linear", dtype="bf16", tokens=1, features=4096, outputs=4096, bias=False),
        # a few sequences generated side by side
        dict(name="linear_f16_few_tokens", kind="linear", dtype="f16", tokens=24, features=4096, outputs=16384, bias=True),
        # a short ragged prompt through a layer of odd width, in full precision
        dict(name="linear_f32_odd", kind="linear", dtype="f32", tokens=197, features=1000, outputs=1003, bias=True),
        # the repository's fully connected benchmark
        dict(name="linear_bf16_large", kind="linear", dtype="bf16", tokens=8192, features=4096, outputs=4096, bias=True),
        # its weight gradient
        dict(name="linear_grad_f16_large", kind="linear_grad", dtype="f16", tokens=8192, features=4096, outputs=4096),
        # the classifier of a small network at a ragged batch
        dict(name="linear_grad_bf16_odd", kind="linear_grad", dtype="bf16", tokens=1000, features=784, outputs=100),
        # one large image served
        dict(name="norm_bf16_one_image", kind="norm", dtype="bf16", n=1, c=512, h=112, w=112, groups=32, activation="silu"),
        # odd planes in full precision, no activation
        dict(name="norm_f32_odd", kind="norm", dtype="f32", n=5, c=96, h=55, w=55, groups=6, activation=None),
        # a training step at the first stage of the repository's benchmark network
        dict(name="norm_train_bf16_large", kind="norm_train", dtype="bf16", n=128, c=256, h=56, w=56, groups=32,
             activation="silu"),
        # a training step of small planes whose groups are no whole vectors
        dict(name="norm_train_f16_small", kind="norm_train", dtype="f16", n=4, c=320, h=16, w=16, groups=32,
             activation="silu"),
    ]


# ------------------------------------------------------------------------------------------
# drawn cases: the same kinds over their ranges
# ------------------------------------------------------------------------------------------
MOST_PRODUCTS = 8192 * 4096 * 4096
MOST_TOKEN_VALUES = 8192 * 4096
MOST_NORM_VALUES = 128 * 256 * 56 * 56


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: half of them whole multiples of 64, half anything."""
    w = _log_int(rng, lo, hi)
    return max(64, w // 64 * 64) if rng.random() < 0.5 else w


def draw(rng):
    kind = rng.choice(["checkpoint", "linear", "linear", "linear_grad", "norm", "norm_train"])
    case = dict(kind=kind, dtype=rng.choice(["f32", "f16", "bf16", "bf16"]))
    if kind == "checkpoint":
        case["tokens"], case["features"] = _log_int(rng, 1, 8192), _width(rng, 16, 16384)
        case["tokens"] = max(1, min(case["tokens"], MOST_TOKEN_VALUES // (2 if case["dtype"] == "f32" else 1) // case["features"]))
    elif kind == "linear":
        case["tokens"], case["features"], case["outputs"] = _log_int(rng, 1, 8192), _width(rng, 32, 16384), _width(rng, 16, 16384)
        case["tokens"] = max(1, min(case["tokens"], MOST_PRODUCTS // (2 * case["features"] * case["outputs"])))
        case["bias"] = rng.random() < 0.5
    elif kind == "linear_grad":
        case["dtype"] = rng.choice(["f16", "bf16"])
        case["tokens"], case["features"], case["outputs"] = _log_int(rng, 16, 8192), _width(rng, 32, 8192), _width(rng, 10, 8192)
        case["tokens"] = max(1, min(case["tokens"], MOST_PRODUCTS // (2 * case["features"] * case["outputs"])))
    else:
        case["groups"] = rng.choice([1, 2, 3, 4, 6, 8, 16, 24, 32, 32])
        case["c"] = case["groups"] * max(1, _log_int(rng, 16, 1024) // case["groups"])
        case["h"] = _log_int(rng, 1, 128)
        case["w"] = case["h"] if rng.random() < 0.6 else max(1, int(case["h"] * rng.uniform(0.6, 1.8)))
        case["n"] = _log_int(rng, 1, 256)
        most = MOST_NORM_VALUES // (4 if case["dtype"] == "f32" else 2)
        case["n"] = max(1, min(case["n"], most // (case["c"] * case["h"] * case["w"])))
        case["activation"] = rng.choice(["silu", "silu", None])
    return case


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _tokens(gen, tokens, features, dtype):
    """Hidden states: their size differs from token to token, a few features are far larger than the others, and a
    padded token is zero."""
    size = torch.randn(tokens, 1, generator=gen, device=DEVICE).mul_(0.5).exp_()
    wide = 1.0 + 7.0 * (torch.rand(1, features, generator=gen, device=DEVICE) < 0.01).float()
    x = torch.randn(tokens, features, generator=gen, device=DEVICE) * size * wide
    if tokens > 8:
        x[torch.rand(tokens, generator=gen, device=DEVICE) < 0.03] = 0.0
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    kind = case["kind"]
    state = dict(case=case)
    if kind in ("norm", "norm_train"):
        n, c, h, w = (case[k] for k in "nchw")
        shape = (n, c, 1, 1)
        x = torch.randn(n, c, h, w, generator=gen, device=DEVICE).to(memory_format=torch.channels_last)
        x = x * torch.randn(shape, generator=gen, device=DEVICE).mul_(0.4).exp_() + 0.3 * torch.randn(shape, generator=gen, device=DEVICE)
        state["x"] = x.to(dtype).contiguous(memory_format=torch.channels_last)
        state["weight"] = 1.0 + 0.2 * torch.randn(c, generator=gen, device=DEVICE)
        state["bias"] = 0.2 * torch.randn(c, generator=gen, device=DEVICE)
        if kind == "norm_train":
            g = torch.randn(n, c, h, w, generator=gen, device=DEVICE).to(dtype)
            state["grad"] = g.contiguous(memory_format=torch.channels_last)
        return state
    x = _tokens(gen, case["tokens"], case["features"], dtype)
    if kind == "linear_grad":
        codes, state["scale"] = _codes(x)
        state["codes"] = _rows_of_16_bytes(codes)
        state["grad"] = torch.randn(case["tokens"], case["outputs"], generator=gen, device=DEVICE).mul_(0.05).to(dtype)
        return state
    state["x"] = x
    if kind == "linear":
        weight = torch.randn(case["outputs"], case["features"], generator=gen, device=DEVICE) / math.sqrt(case["features"])
        codes, state["weight_scale"] = _codes(weight)
        state["weight_codes"] = _rows_of_16_bytes(codes)
        state["bias"] = 0.1 * torch.randn(case["outputs"], generator=gen, device=DEVICE) if case["bias"] else None
    return state


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
def _scaled(x, largest):
    """127 x / largest, rounded, halves away from zero: in 64 bits, values next to a half decide a code."""
    largest = largest.double()
    t = torch.where(largest >= SMALLEST, 127.0 * x.double() / largest, 0.0)
    return torch.copysign(torch.floor(t.abs() + 0.5), t)


def _rows_of_16_bytes(codes):
    """The same codes in rows that begin at multiples of 16 bytes, as the framework lays them out."""
    features = codes.shape[1]
    kept = codes.new_zeros(codes.shape[0], (features + 15) // 16 * 16)
    kept[:, :features] = codes
    return kept[:, :features]


def _codes(x):
    """int8 codes [tokens, features] and 32-bit scales [tokens] of the rows of x."""
    largest = x.float().abs().amax(dim=-1, keepdim=True)
    scale = torch.where(largest >= SMALLEST, largest / 127.0, 0.0)
    return _scaled(x, largest).to(torch.int8), scale.squeeze(-1)


def _plain_norm(state, train):
    case, x = state["case"], state["x"]
    n, c, h, w = x.shape
    groups, silu = case["groups"], case["activation"] == "silu"
    rows = x.permute(0, 2, 3, 1).reshape(n, h * w, groups, c // groups).float()
    weight, bias = state["weight"].view(groups, -1), state["bias"].view(groups, -1)
    mean = rows.mean(dim=(1, 3), keepdim=True)
    rstd = (rows - mean).square().mean(dim=(1, 3), keepdim=True).add(EPS).rsqrt()
    z = (rows - mean) * rstd * weight + bias
    y = z * torch.sigmoid(z) if silu else z

    def images(t):
        return t.to(x.dtype).view(n, h, w, c).permute(0, 3, 1, 2)

    if not train:
        return images(y)
    largest = rows.abs().amax(dim=(1, 3), keepdim=True)
    scale = torch.where(largest >= SMALLEST, largest / 127.0, 0.0)
    kept = _scaled(rows, largest).float() * scale
    normal = (kept - mean) * rstd
    grad = state["grad"].permute(0, 2, 3, 1).reshape(rows.shape).float()
    if silu:
        z = normal * weight + bias
        s = torch.sigmoid(z)
        grad = grad * s * (1.0 + z * (1.0 - s))
    grad_bias = grad.sum(dim=(0, 1)).view(-1)
    grad_weight = (grad * normal).sum(dim=(0, 1)).view(-1)
    inner = grad * weight
    first = inner.mean(dim=(1, 3), keepdim=True)
    second = (inner * normal).mean(dim=(1, 3), keepdim=True)
    return images(y), images(rstd * (inner - first - normal * second)), grad_weight, grad_bias


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _own(state)
    if kind == "checkpoint":
        codes, scale = _codes(state["x"])
        return (codes.float() * scale[:, None]).to(state["x"].dtype), scale
    if kind == "linear":
        codes, scale = _codes(state["x"])
        y = torch.matmul(codes.float(), state["weight_codes"].float().t()) * scale[:, None] * state["weight_scale"]
        return (y if state["bias"] is None else y + state["bias"]).to(state["x"].dtype)
    if kind == "linear_grad":
        kept = state["codes"].float() * state["scale"][:, None]
        return torch.matmul(state["grad"].float().t(), kept).to(state["grad"].dtype)
    return _plain_norm(state, kind == "norm_train")


def _own(state):
    from actnn_amd.cpp_extension import backward_func, tokens
    case = state["case"]
    kind = case["kind"]
    if kind == "checkpoint":
        codes, scale = tokens.quantize_tokens(state["x"])
        return tokens.dequantize_tokens(codes, scale, state["x"].dtype), scale
    if kind == "linear":
        return tokens.linear_tokens(state["x"], state["weight_codes"], state["weight_scale"], state["bias"])
    if kind == "linear_grad":
        return tokens.linear_tokens_grad_weight(state["grad"], state["codes"], state["scale"])
    groups, activation = case["groups"], case["activation"]
    if kind == "norm":
        return backward_func.hip_group_norm_forward(state["x"], groups, state["weight"], state["bias"], EPS, activation)[0]
    output, mean, rstd, codes, scale = backward_func.hip_group_norm_forward(
        state["x"], groups, state["weight"], state["bias"], EPS, activation, keep=True)
    return (output,) + tuple(backward_func.hip_group_norm_backward(
        state["grad"], codes, scale, groups, state["weight"], state["bias"], mean, rstd, activation))


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------
def _exact_rows(x, dims):
    """What the 8-bit codes of x stand for, one scale over `dims`."""
    x = x.double()
    top = x.abs().amax(dim=dims, keepdim=True)
    top = torch.where(top < SMALLEST, torch.zeros_like(top), top)
    part = torch.where(top > 0, x / torch.where(top > 0, top, torch.ones_like(top)), torch.zeros_like(x))
    # 127 * part rounded: x is at most `top`, so the doubled value's whole part tells the side of the half
    twice = torch.trunc((254.0 * x.abs()) / torch.where(top > 0, top, torch.ones_like(top)))
    code = torch.trunc((twice + 1.0) / 2.0) * torch.sign(part)
    return code * (top / 127.0), top / 127.0


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "checkpoint":
        values, scale = _exact_rows(state["x"], (1,))
        return values, scale[:, 0]
    if kind == "linear":
        values, _ = _exact_rows(state["x"], (1,))
        y = values @ (state["weight_codes"].double() * state["weight_scale"].double().unsqueeze(1)).t()
        return y + state["bias"].double() if state["bias"] is not None else y
    if kind == "linear_grad":
        return (state["grad"].double() * state["scale"].double().unsqueeze(1)).t() @ state["codes"].double()
    x, groups, c = state["x"].double(), case["groups"], case["c"]
    shape = x.shape
    x = x.reshape(shape[0], groups, -1)
    count = x.shape[2]
    mean = x.sum(dim=2, keepdim=True) / count
    centred = x - mean
    spread = torch.sqrt((centred * centred).sum(dim=2, keepdim=True) / count + EPS)
    weight, bias = state["weight"].double().view(1, c, 1, 1), state["bias"].double().view(1, c, 1, 1)
    z = (centred / spread).view(shape) * weight + bias
    silu = case["activation"] == "silu"
    y = z / (1.0 + torch.exp(-z)) if silu else z
    if kind == "norm":
        return y
    kept, _ = _exact_rows(x, (2,))
    normal = ((kept - mean) / spread).view(shape)
    slope = state["grad"].double()
    if silu:
        z = normal * weight + bias
        e = torch.exp(-z)
        slope = slope * ((1.0 + e + z * e) / (1.0 + e) ** 2)
    by_normal = slope * normal
    grad_weight, grad_bias = by_normal.sum(dim=(0, 2, 3)), slope.sum(dim=(0, 2, 3))
    inner = (slope * weight).reshape(shape[0], groups, -1)
    normal = normal.reshape(shape[0], groups, -1)
    grad_x = (inner - inner.mean(dim=2, keepdim=True) - normal * (inner * normal).mean(dim=2, keepdim=True)) / spread
    return y, grad_x.view(shape), grad_weight, grad_bias


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    """Bytes: each input once, each output once (and, where a pass keeps 8 bits in between, those written and read
    once).  Operations: two for each product of a matrix product, a few for each value of the others."""
    kind, size = case["kind"], BYTES[case["dtype"]]
    if kind in ("norm", "norm_train"):
        values = case["n"] * case["c"] * case["h"] * case["w"]
        if kind == "norm":
            return dict(bytes=2 * size * values + 8 * case["c"], flops=8 * values)
        return dict(bytes=(4 * size + 2) * values + 16 * case["c"], flops=30 * values)
    tokens, features = case["tokens"], case["features"]
    if kind == "checkpoint":
        return dict(bytes=(2 * size + 2) * tokens * features + 8 * tokens, flops=4 * tokens * features)
    outputs = case["outputs"]
    if kind == "linear":
        return dict(bytes=size * tokens * (features + outputs) + outputs * (features + 4 + (4 if case["bias"] else 0)),
                    flops=2 * tokens * features * outputs)
    return dict(bytes=size * tokens * outputs + tokens * (features + 4) + size * outputs * features,
                flops=2 * tokens * features * outputs)
