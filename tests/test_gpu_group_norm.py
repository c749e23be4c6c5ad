"""Group norm with its activation, channels last, forward and backward, against the formulas in 64 bits."""
import pytest
import torch

from actnn_amd.cpp_extension import backward_func as bf
from oracle import group_norm as oracle

DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}       # half of the smallest step
# Additions in a row that a sum is made of: 32 about one value, at most 256 rows of threads, 64 slices, 64 lanes' steps: below 512,
# each rounding to 2^-24 of what has been summed.
SUMMED = 2.0 ** -15


def channels_last(t):
    order = [0] + list(range(2, t.dim())) + [1]
    back = [0, t.dim() - 1] + list(range(1, t.dim() - 1))
    return t.permute(order).contiguous().permute(back)


def make(shape, dtype, seed, affine=True, spread=0.4):
    gen = torch.Generator().manual_seed(seed)
    C = shape[1]
    by = (shape[0], C) + (1,) * (len(shape) - 2)
    x = torch.randn(shape, generator=gen) * torch.exp(spread * torch.randn(by, generator=gen)) + 0.5 * torch.randn(by, generator=gen)
    dy = torch.randn(shape, generator=gen)
    w = 1 + 0.3 * torch.randn(C, generator=gen) if affine else None
    b = 0.3 * torch.randn(C, generator=gen) if affine else None
    put = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    return channels_last(x.to(dtype).to(DEV)), channels_last(dy.to(dtype).to(DEV)), put(w), put(b)


def along(t, x, groups):
    """[N, G] to the shape of x."""
    N, C = x.shape[:2]
    return t[:, :, None].expand(N, groups, C // groups).reshape((N, C) + (1,) * (x.dim() - 2)).double()


def by_channel(t, x, empty):
    return empty if t is None else t.double().view((1, -1) + (1,) * (x.dim() - 2))


def check_forward(x, groups, w, b, eps, activation, got):
    y, mean, rstd, codes, scale = got
    exact, m, r = oracle.forward(x, groups, w, b, eps, activation)
    top = x.double().abs().reshape(x.shape[0], groups, -1).amax(2)
    spread = (x.double().reshape(x.shape[0], groups, -1) - m[:, :, None]).abs().amax(2)
    # sums about a value of the group: their terms are at most twice the spread; the mean itself is rounded
    off_mean = SUMMED * 2 * spread + 2.0 ** -22 * m.abs()
    assert mean.shape == rstd.shape == m.shape
    assert ((mean.double() - m).abs() <= off_mean + 1e-37).all()
    # the variance: sums of positive terms about a mean that is off by off_mean; rstd has half its relative error
    off_rstd = r * (SUMMED + (off_mean * r) ** 2 + 2 * 2.0 ** -22)
    assert ((rstd.double() - r).abs() <= off_rstd).all()
    wa, ba = by_channel(w, x, 1.0), by_channel(b, x, 0.0)
    n = (x.double() - along(m, x, groups)) * along(r, x, groups)
    z = n * wa + ba
    off = abs(wa) * (along(off_mean * r, x, groups) + n.abs() * along(off_rstd / r, x, groups)) + 2.0 ** -22 * ((n * wa).abs() + abs(ba))
    if activation == "silu":
        # the slope of z sigmoid(z) is at most 1.1; the sigmoid's exponent is rounded to 2^-24 of itself
        off = 1.1 * off + 2.0 ** -22 * (2 + z.abs()) * exact.abs()
    assert y.dtype == x.dtype and y.shape == x.shape
    assert ((y.double() - exact).abs() <= off + HALF_STEP[x.dtype] * exact.abs() + TINY[x.dtype]).all()
    if x.dtype == torch.float32 and x.numel() > 1000 and float((top / spread.clamp(min=1e-30)).max()) < 100:
        assert (y.double() - exact).norm() <= 2.0 ** -20 * exact.norm()
    if codes is not None:
        q, s = oracle.kept(x, groups)
        assert codes.dtype == torch.int8 and torch.equal(codes.cpu().double(), q)
        assert ((scale.cpu().double() - s).abs() <= 2.0 ** -24 * s).all()


def check_backward(dy, values, mean, rstd, groups, w, b, activation, got):
    dx, dw, db = got
    ex, ew, eb = oracle.backward(dy, values, mean, rstd, groups, w, b, activation)
    wa, ba = by_channel(w, dy, torch.ones(1, device=DEV, dtype=torch.float64)), by_channel(b, dy, 0.0)
    N, C = dy.shape[:2]
    dims = [0] + list(range(2, dy.dim()))
    m, r = along(mean, dy, groups), along(rstd, dy, groups)
    n = (values.double() - m) * r
    off_n = 2.0 ** -22 * (values.double().abs() + m.abs()) * r
    z = n * wa + ba
    off_z = off_n * wa.abs() + 2.0 ** -23 * (z.abs() + abs(ba))
    dz, off_dz = dy.double(), torch.zeros_like(z)
    if activation == "silu":
        s = torch.sigmoid(z)
        slope = s * (1 + z * (1 - s))
        # the slope's own slope is at most 1/2; its sigmoid as above
        off_dz = dz.abs() * (0.5 * off_z + 2.0 ** -21 * (2 + z.abs()) * s * (1 + z.abs()))
        dz = dz * slope
    size_b, size_w = dz.abs().sum(dims), (dz * n).abs().sum(dims)
    off_b = SUMMED * size_b + off_dz.sum(dims)
    off_w = SUMMED * size_w + (off_dz * n.abs() + dz.abs() * off_n).sum(dims)
    if b is None:
        assert db is None
    else:
        assert ((db.double() - eb).abs() <= off_b + 1e-37).all()
    if w is None:
        assert dw is None
    else:
        assert ((dw.double() - ew).abs() <= off_w + 1e-37).all()

    def group_mean(t):
        return along(t.reshape(N, groups, -1).mean(2), dy, groups)

    u, un = (dz * wa).abs(), (dz * wa * n).abs()
    off_u, off_un = off_dz * wa.abs(), (off_dz * n.abs() + dz.abs() * off_n) * wa.abs()
    off = r * (off_u + group_mean(SUMMED * u + off_u) + n.abs() * group_mean(SUMMED * un + off_un) + off_n * group_mean(un)
               + 2.0 ** -21 * (u + group_mean(u) + n.abs() * group_mean(un)))
    assert dx.dtype == dy.dtype and dx.shape == dy.shape
    assert ((dx.double() - ex).abs() <= off + HALF_STEP[dy.dtype] * ex.abs() + TINY[dy.dtype]).all()


# (shape, groups): aligned vectors, groups narrower than a vector, groups across vectors, odd channel counts (nothing aligned), one
# group, a group per channel, groups wider than a block, one pixel, one value a group, 2-d to 5-d tensors
CASES = [((2, 64, 9, 11), 8), ((3, 320, 16, 16), 32), ((1, 96, 55, 53), 6), ((5, 24, 7, 7), 24), ((4, 32, 5, 3), 16), ((2, 33, 10, 9), 11),
         ((2, 30, 12, 5), 6), ((7, 128, 1, 1), 4), ((3, 6, 4, 4), 3), ((1, 1, 1, 1), 1), ((2, 3, 1, 1), 3), ((130, 64), 8), ((3, 48, 301), 4),
         ((2, 16, 3, 4, 5), 2), ((1, 512, 40, 40), 32), ((2, 5000, 3, 3), 1), ((1, 4999, 2, 5), 1), ((2, 2100, 4, 3), 700), ((1, 6144, 2, 2), 2),
         ((40, 40, 6, 6), 5), ((1, 8, 300, 301), 1), ((300, 16, 2, 2), 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", CASES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_and_backward(shape, groups, dtype):
    for i, activation in enumerate((None, "silu")):
        print(f"[group_norm] {shape} groups {groups} {dtype} {activation}", flush=True)
        x, dy, w, b = make(shape, dtype, sum(shape) + i, affine=(sum(shape) + i) % 3 != 0)
        got = bf.hip_group_norm_forward(x, groups, w, b, 1e-5, activation, keep=True)
        check_forward(x, groups, w, b, 1e-5, activation, got)
        y, mean, rstd, codes, scale = got
        alone = bf.hip_group_norm_forward(x, groups, w, b, 1e-5, activation)
        assert all(torch.equal(p, q) for p, q in zip(got[:3], alone)) and alone[3] is None and alone[4] is None
        values = codes.double() * along(scale, x, groups)
        grads = bf.hip_group_norm_backward(dy, codes, scale, groups, w, b, mean, rstd, activation)
        check_backward(dy, values, mean, rstd, groups, w, b, activation, grads)
        again = bf.hip_group_norm_backward(dy, codes, scale, groups, w, b, mean, rstd, activation)
        assert all(p is q is None or torch.equal(p, q) for p, q in zip(grads, again))
        full = bf.hip_group_norm_backward(dy, None, None, groups, w, b, mean, rstd, activation, input=x)
        check_backward(dy, x, mean, rstd, groups, w, b, activation, full)


# blocks enough for the whole chip: chunks of whole lines in one kernel and in two, whole pixels, groups of a chunk and wider ones
MANY = [((200, 192, 20, 20), 32), ((200, 320, 16, 16), 32), ((130, 1280, 8, 8), 32), ((150, 366, 17, 16), 6), ((60, 770, 14, 14), 1),
        ((300, 100, 9, 11), 20), ((3, 2056, 30, 30), 1), ((1100, 24, 9, 9), 3), ((1, 640, 300, 70), 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", MANY)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_and_backward_of_many_blocks(shape, groups, dtype):
    test_forward_and_backward(shape, groups, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [0, 12345])
def test_statistics_far_from_zero_and_with_an_outlier(dtype, at):
    for shape, groups in (((2, 64, 40, 40), 4), ((1, 30, 61, 50), 3)):
        x, _, w, b = make(shape, torch.float32, 5, spread=0.0)
        far = channels_last((x * (1.0 if dtype == torch.float32 else 8.0) + 1000.0).to(dtype))
        check_forward(far, groups, w, b, 1e-5, None, bf.hip_group_norm_forward(far, groups, w, b, 1e-5, None, keep=True))
        flat = x.permute(0, 2, 3, 1).reshape(-1)
        flat[at] = 30000.0
        out = channels_last(flat.view(shape[0], shape[2], shape[3], shape[1]).permute(0, 3, 1, 2).to(dtype))
        check_forward(out, groups, w, b, 1e-5, "silu", bf.hip_group_norm_forward(out, groups, w, b, 1e-5, "silu", keep=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_zero_and_spoiled_groups(dtype):
    x, dy, w, b = make((3, 32, 6, 6), dtype, 8)
    x[0, :8] = 0
    x[1, 8:16] = 3.0
    got = bf.hip_group_norm_forward(x, 4, w, b, 1e-5, None, keep=True)
    check_forward(x, 4, w, b, 1e-5, None, got)
    y, mean, rstd, codes, scale = got
    assert (codes[0, :8] == 0).all() and scale[0, 0] == 0
    # the parameters' gradients of every other sample and channel are untouched by a spoiled group, the group's own say so
    x[2, 16, 3, 3] = float("nan")
    x[2, 24, 0, 0] = float("inf")
    y2, mean2, rstd2, codes2, scale2 = bf.hip_group_norm_forward(x, 4, w, b, 1e-5, None, keep=True)
    assert torch.isnan(y2[2, 16:]).all() and torch.isnan(scale2[2, 2:]).all() and (codes2[2, 16:] == 0).all()
    assert torch.equal(y2[2, :16], y[2, :16]) and torch.equal(y2[:2], y[:2])
    dx, dw, db = bf.hip_group_norm_backward(dy, codes2, scale2, 4, w, b, mean2, rstd2)
    dx1, dw1, db1 = bf.hip_group_norm_backward(dy, codes, scale, 4, w, b, mean, rstd)
    assert torch.isnan(dx[2, 16:]).all() and torch.equal(dx[:2], dx1[:2]) and torch.equal(dw[:16], dw1[:16]) and torch.equal(db, db1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_and_layouts(dtype):
    x, dy, w, b = make((2, 40, 9, 7), dtype, 2)
    want = bf.hip_group_norm_forward(x, 5, w, b, 1e-5, "silu", keep=True)
    # the same values at an address that is a multiple of the element only
    room = torch.zeros(x.numel() + 3, dtype=dtype, device=DEV)
    odd = room[3:].view(2, 9, 7, 40).permute(0, 3, 1, 2)
    odd.copy_(x)
    got = bf.hip_group_norm_forward(odd, 5, w, b, 1e-5, "silu", keep=True)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    args = (5, w, b, want[1], want[2], "silu")
    grads = bf.hip_group_norm_backward(dy, want[3], want[4], *args)
    for g in (dy.contiguous(), dy.transpose(2, 3).contiguous().transpose(2, 3)):
        assert all(torch.equal(p, q) for p, q in zip(grads, bf.hip_group_norm_backward(g, want[3].contiguous(), want[4], *args)))
    even = dy[:, :, :1, :1].expand(2, 40, 9, 7)
    assert torch.equal(bf.hip_group_norm_backward(even, want[3], want[4], *args)[0],
                       bf.hip_group_norm_backward(channels_last(even), want[3], want[4], *args)[0])
    half = bf.hip_group_norm_forward(x, 5, w.bfloat16(), b.half(), 1e-5, "silu")           # parameters of other types
    assert torch.equal(half[0], bf.hip_group_norm_forward(x, 5, w.bfloat16().float(), b.half().float(), 1e-5, "silu")[0])
    if x.is_contiguous(memory_format=torch.channels_last):
        assert want[0].is_contiguous(memory_format=torch.channels_last) and grads[0].is_contiguous(memory_format=torch.channels_last)


@pytest.mark.gpu
def test_nothing_behind_the_tensors_is_written(lib):
    N, C, P, G = 2, 21, 15, 3
    x = torch.randn(N, P, C, device=DEV).bfloat16()
    y = torch.full((N * P * C + 16,), 5.0, device=DEV, dtype=torch.bfloat16)
    codes = torch.full((N * P * C + 16,), 77, device=DEV, dtype=torch.int8)
    mean, rstd, scale = (torch.full((N * G + 4,), 9.0, device=DEV) for _ in range(3))
    stream = torch.cuda.current_stream().cuda_stream
    for backward in (0, 1):
        bytes_ = lib.actnn_group_norm_workspace_bytes(N, C, P, G, 2, backward)
        ws = torch.full((bytes_ + 64,), 33, dtype=torch.uint8, device=DEV)
        if not backward:
            rc = lib.actnn_group_norm_forward(x.data_ptr(), None, None, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), codes.data_ptr(),
                                              scale.data_ptr(), N, C, P, G, 1e-5, 1, 2, ws.data_ptr(), bytes_, stream)
        else:
            dw, db = (torch.full((C + 4,), 9.0, device=DEV) for _ in range(2))
            rc = lib.actnn_group_norm_backward(x.data_ptr(), codes.data_ptr(), scale.data_ptr(), None, None, None, mean.data_ptr(),
                                               rstd.data_ptr(), y.data_ptr(), dw.data_ptr(), db.data_ptr(), N, C, P, G, 1, 2,
                                               ws.data_ptr(), bytes_, stream)
            assert (dw[C:] == 9).all() and (db[C:] == 9).all()
        assert rc == 0 and (ws[bytes_:] == 33).all() and (y[N * P * C:] == 5).all() and (codes[N * P * C:] == 77).all()
        assert all((t[N * G:] == 9).all() for t in (mean, rstd, scale))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    # 2.2e9 values in one sample, and in many: the last group, the last sample are what they are by themselves
    x = torch.zeros(1, 6000, 6000, 64, dtype=torch.bfloat16, device=DEV).permute(0, 3, 1, 2)
    last = torch.randn(1, 8, 6000, 6000, device=DEV).bfloat16()
    x[:, 56:] = last
    y, mean, rstd, codes, scale = bf.hip_group_norm_forward(x, 8, None, None, 1e-5, "silu", keep=True)
    v = last.double()
    m, var = v.mean(), v.var(unbiased=False)
    assert abs(mean[0, 7].item() - m.item()) < 1e-5 and abs(rstd[0, 7].item() - (var + 1e-5).rsqrt().item()) < 1e-5
    z = (v[0, :, -3:] - m) * (var + 1e-5).rsqrt()
    exact = z * torch.sigmoid(z)
    assert ((y[0, 56:, -3:].double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 1e-4).all() and not y[:, :56].any()
    assert torch.equal(codes[0, 56:, -3:].cpu().double(), oracle.kept(last, 1)[0][0, :, -3:])
    dx, _, _ = bf.hip_group_norm_backward(y, codes, scale, 8, None, None, mean, rstd, "silu")
    assert not dx[:, :56].any() and dx[0, 56:, -1].abs().max() > 0.1
    del dx, y, codes, v, last, z, x
    x = torch.zeros(8400, 16, 16, 1024, dtype=torch.float16, device=DEV).permute(0, 3, 1, 2)
    x[-1] = torch.randn(1024, 16, 16, device=DEV)
    y = bf.hip_group_norm_forward(x, 32, None, None, 1e-5)[0]
    assert torch.equal(y[-1:], bf.hip_group_norm_forward(x[-1:], 32, None, None, 1e-5)[0]) and not y[:-1].any()


@pytest.mark.gpu
def test_empty_tensors():
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4)):
        x = torch.zeros(shape, device=DEV)
        w = torch.ones(8, device=DEV)
        y, mean, rstd, codes, scale = bf.hip_group_norm_forward(x, 2, w, w, 1e-5, "silu", keep=True)
        assert y.shape == codes.shape == shape and mean.shape == (shape[0], 2)
        dx, dw, db = bf.hip_group_norm_backward(x, codes, scale, 2, w, w, mean, rstd, "silu")
        assert dx.shape == shape and (dw == 0).all() and (db == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 64, 32, 32), 8), ((3, 30, 5, 7), 6)])
def test_captured_and_replayed(shape, groups):
    x, dy, w, b = make(shape, torch.bfloat16, 4)

    def step():
        y, mean, rstd, codes, scale = bf.hip_group_norm_forward(x, groups, w, b, 1e-5, "silu", keep=True)
        return (y,) + tuple(bf.hip_group_norm_backward(dy, codes, scale, groups, w, b, mean, rstd, "silu"))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(torch.randn(shape, device=DEV) * (i + 1))
        dy.copy_(torch.randn(shape, device=DEV))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), i


def test_refusals_on_the_cpu():
    x = torch.zeros(2, 8, 3, 3).contiguous(memory_format=torch.channels_last)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        bf.hip_group_norm_forward(x, 2, None, None, 1e-5)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        bf.hip_group_norm_backward(x, x.to(torch.int8), torch.zeros(2, 2), 2, None, None, torch.zeros(2, 2), torch.zeros(2, 2))
    with pytest.raises(RuntimeError, match="None or 'silu'"):
        bf.hip_group_norm_forward(x, 2, None, None, 1e-5, "relu")


@pytest.mark.gpu
def test_refusals():
    x, dy, w, b = make((2, 8, 3, 5), torch.float32, 1)
    f, g = bf.hip_group_norm_forward, bf.hip_group_norm_backward
    for args, text in (((x.contiguous(), 2, w, b, 1e-5), "channels last"), ((x, 3, w, b, 1e-5), "multiple of the groups"), ((x, 0, w, b, 1e-5), "groups"),
                       ((x.double(), 2, w, b, 1e-5), "type of input"), ((x, 2, w[:7], b, 1e-5), "one value for each channel"),
                       ((x, 2, w, b.cpu(), 1e-5), "CUDA"), ((x[:, 0, 0, 0], 2, w, b, 1e-5), "dimension")):
        with pytest.raises(RuntimeError, match=text):
            f(*args)
    y, mean, rstd, codes, scale = f(x, 2, w, b, 1e-5, None, True)
    good = [dy, codes, scale, 2, w, b, mean, rstd]
    for i, bad, text in ((0, dy[:1], "same shape"), (1, codes.float(), "type of codes"), (1, None, "either"), (2, scale[:1], "one value for each row"),
                         (6, mean[:1], "one value for each row"), (7, rstd.double(), "type of rstd"), (3, 3, "multiple of the groups"),
                         (0, dy.to(torch.int32), "type of grad_output"), (1, codes.cpu(), "CUDA")):
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError, match=text):
            g(*args)
    with pytest.raises(RuntimeError, match="either"):
        g(*good, input=x)


def test_c_abi_refuses_bad_sizes(lib):
    ws, f, g = lib.actnn_group_norm_workspace_bytes, lib.actnn_group_norm_forward, lib.actnn_group_norm_backward
    assert ws(2, 64, 100, 8, 2, 0) > 0 and ws(2, 64, 100, 8, 2, 1) > 0
    assert ws(2, 64, 100, 7, 2, 0) == -1 and ws(2, 64, 100, 8, 5, 0) == -2 and ws(0, 64, 100, 8, 2, 0) == 0
    none = [None] * 8
    assert f(*none, 2, 64, 100, 7, 1e-5, 0, 2, None, 0, None) == -1
    assert f(*none, 2, 64, 100, 8, 1e-5, 2, 2, None, 0, None) == -1           # unknown activation
    assert f(*none, 2, 64, 100, 8, 1e-5, 0, 2, None, 0, None) == -1           # null pointers
    assert f(*none, 0, 64, 100, 8, 1e-5, 0, 2, None, 0, None) == 0
    at = [16, None, None, 16, 16, 16, None, None]
    assert f(*at, 2, 64, 100, 8, 1e-5, 0, 2, 16, 8, None) == -1               # workspace too small
    assert f(*at, 2, 64, 100, 8, 1e-5, 0, 2, 8, 1 << 20, None) == -4
    assert f(*at, 0x7fffff, 4096, 1, 32, 1e-5, 0, 2, 16, 1 << 60, None) == -1 # more blocks than a launch takes
    assert g(*[None] * 11, 2, 64, 100, 8, 0, 2, None, 0, None) == -1
    assert g(*[None] * 11, 2, 64, 100, 8, 0, 9, None, 0, None) == -2
