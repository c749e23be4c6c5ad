"""The product in 8-bit integers against the same sum in 64 bits, and linear_tokens against its two steps."""
import pytest
import torch

from actnn_amd.cpp_extension import tokens

DEV = "cuda:0"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}       # half of fp16's smallest step


def make(M, K, O, seed, bias):
    gen = torch.Generator().manual_seed(seed)

    def codes(n):
        return torch.randint(-127, 128, (n, K), generator=gen, dtype=torch.int32).to(torch.int8)

    scale = torch.rand(M, generator=gen) * 0.01 / 127
    wscale = torch.rand(O, generator=gen) / 127
    return codes(M), scale, codes(O), wscale, torch.randn(O, generator=gen) if bias else None


def laid(codes, fill=None):
    """Rows at multiples of 16 bytes; what lies between them is `fill`."""
    M, K = codes.shape
    room = torch.zeros(M, (K + 15) // 16 * 16, dtype=torch.int8, device=DEV)
    if fill is not None:
        room.fill_(fill)
    room[:, :K] = codes.to(DEV)
    return room[:, :K]


def check(y, codes, scale, wcodes, wscale, bias, dtype):
    product = (codes.to(DEV).double() @ wcodes.to(DEV).double().t()) * scale.to(DEV).double()[:, None] * wscale.to(DEV).double()
    exact = product if bias is None else product + bias.to(DEV).double()
    assert y.dtype == dtype and y.shape == exact.shape
    # the sum's conversion and two products round to 32 bits, then the addition, then the output
    bound = 3.01 * 2.0 ** -24 * product.abs() + (2.0 ** -24 + HALF_STEP[dtype]) * exact.abs() * 1.001 + SMALLEST[dtype]
    err = (y.double() - exact).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


# few tokens in one to four tiles of 16; tiles of 64 (by 64 and 128 features) with and without slices, of 128 and of 256; odd everything
SHAPES = [(1, 1, 1), (1, 16, 16), (1, 4096, 300), (2, 100, 17), (3, 1003, 33), (15, 64, 64), (16, 65, 1), (17, 128, 130), (24, 4100, 257),
          (32, 31, 16), (33, 513, 100), (64, 1000, 1003), (65, 15, 3), (65, 8192, 70), (100, 16, 64), (128, 128, 128), (129, 129, 65),
          (197, 1000, 1003), (70, 5000, 4), (300, 2000, 301), (1100, 257, 2100), (2048, 144, 2050), (2048, 200, 8192), (4100, 272, 4100), (66, 127, 20000), (130, 2048, 2000),
          (256, 2100, 4096), (100, 8200, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,O", SHAPES)
def test_product(M, K, O):
    for i, dtype in enumerate((torch.float32, torch.float16, torch.bfloat16)):
        print(f"[tokens_matmul] {M}x{K}x{O} {dtype}", flush=True)
        codes, scale, wcodes, wscale, bias = make(M, K, O, M + K + O + i, bias=i != 1)
        y = tokens.matmul_tokens(laid(codes, 99), scale.to(DEV), laid(wcodes, -77), wscale.to(DEV), None if bias is None else bias.to(DEV), dtype)
        check(y, codes, scale, wcodes, wscale, bias, dtype)


# few tokens by tiles, with slices of any number; tiles whose last round is half empty
@pytest.mark.gpu
@pytest.mark.parametrize("M,K,O", [(5, 16384, 100), (16, 2048, 16400), (24, 4090, 16390), (31, 12300, 70), (33, 512, 40), (48, 9001, 200), (61, 7326, 1790),
                                   (500, 6100, 450), (700, 14208, 130), (2300, 1024, 1030), (1351, 3000, 720)])
def test_product_between_the_kernels(M, K, O):
    test_product(M, K, O)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 20, 65, 300])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_sums(M, sign):
    K, O = 131071, 5
    codes = torch.full((M, K), -128, dtype=torch.int8)
    wcodes = torch.full((O, K), -128 if sign > 0 else 127, dtype=torch.int8)
    one = torch.ones(M), torch.ones(O)
    y = tokens.matmul_tokens(laid(codes), one[0].to(DEV), laid(wcodes), one[1].to(DEV))
    check(y, codes, one[0], wcodes, one[1], None, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,O", [(1, 64, 40), (1, 4096, 50), (1, 24, 17), (2, 1000, 33), (3, 1003, 16), (4, 4104, 100), (4, 16384, 20), (4, 16392, 20),
                                   (5, 256, 48), (9, 1003, 130), (70, 200, 70), (600, 1030, 250)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_linear_is_its_two_steps(M, K, O, dtype):
    gen = torch.Generator().manual_seed(M)
    x = (torch.randn(M, K, generator=gen) * 3).to(dtype).to(DEV)
    if M > 5:
        x[4] = 0
    wcodes, wscale = tokens.quantize_tokens(torch.randn(O, K, generator=gen).to(DEV))
    for bias in (None, torch.randn(O, generator=gen).to(DEV), torch.randn(O, generator=gen).to(dtype).to(DEV)):
        y, codes, scale = tokens.linear_tokens(x, wcodes, wscale, bias, keep=True)
        c2, s2 = tokens.quantize_tokens(x)
        assert torch.equal(codes, c2) and torch.equal(scale, s2)
        assert torch.equal(y, tokens.matmul_tokens(codes, scale, wcodes, wscale, bias, dtype))
        assert torch.equal(y, tokens.linear_tokens(x, wcodes, wscale, bias))
        check(y, codes.cpu(), scale.cpu(), wcodes.cpu(), wscale.cpu(), None if bias is None else bias.float().cpu(), dtype)
    if M > 5:
        assert torch.equal(y[4], bias.to(dtype))                        # a padded token gives the bias


@pytest.mark.gpu
def test_a_bad_token_spoils_its_own_row_only():
    for M in (4, 5, 300):
        x = torch.randn(M, 100, device=DEV)
        wcodes, wscale = tokens.quantize_tokens(torch.randn(70, 100, device=DEV))
        clean = tokens.linear_tokens(x, wcodes, wscale)
        x[1, 50], x[3, 0] = float("nan"), float("-inf")
        y = tokens.linear_tokens(x, wcodes, wscale)
        assert torch.isnan(y[[1, 3]]).all()
        rest = [i for i in range(M) if i not in (1, 3)]
        assert torch.equal(y[rest], clean[rest])


@pytest.mark.gpu
def test_layouts_and_leading_dimensions():
    codes, scale, wcodes, wscale, bias = make(30, 90, 50, 1, True)
    base = tokens.matmul_tokens(laid(codes), scale.to(DEV), laid(wcodes), wscale.to(DEV), bias.to(DEV))
    assert torch.equal(base, tokens.matmul_tokens(codes.to(DEV), scale.to(DEV), wcodes.to(DEV).t().contiguous().t(), wscale.to(DEV), bias.to(DEV)))
    wide = torch.zeros(30, 256, dtype=torch.int8, device=DEV)
    wide[:, 32:122] = codes.to(DEV)
    assert torch.equal(base, tokens.matmul_tokens(wide[:, 32:122], scale.to(DEV), laid(wcodes), wscale.to(DEV), bias.to(DEV)))
    y = tokens.matmul_tokens(laid(codes).unflatten(0, (5, 6)), scale.to(DEV).view(5, 6), laid(wcodes), wscale.to(DEV), bias.to(DEV))
    assert y.shape == (5, 6, 50) and torch.equal(y.view(30, 50), base)
    y = tokens.matmul_tokens(laid(codes)[7], scale.to(DEV)[7], laid(wcodes), wscale.to(DEV), bias.to(DEV))
    assert y.shape == (50,) and torch.equal(y, base[7])
    assert tokens.matmul_tokens(laid(codes)[:0], scale.to(DEV)[:0], laid(wcodes), wscale.to(DEV)).shape == (0, 50)
    assert tokens.linear_tokens(torch.zeros(3, 90, device=DEV), laid(wcodes)[:0], wscale.to(DEV)[:0]).shape == (3, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,O", [(1, 2048, 512), (40, 515, 100), (70, 4096, 64), (300, 600, 300)])
def test_captured_and_replayed(M, K, O):
    x = torch.randn(M, K, device=DEV).bfloat16()
    wcodes, wscale = tokens.quantize_tokens(torch.randn(O, K, device=DEV))
    bias = torch.randn(O, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tokens.linear_tokens(x, wcodes, wscale, bias)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tokens.linear_tokens(x, wcodes, wscale, bias)
    for i in range(4):
        x.copy_(torch.randn(M, K, device=DEV).bfloat16() * (i + 1))
        graph.replay()
        want = tokens.linear_tokens(x, wcodes, wscale, bias)
        torch.cuda.synchronize()
        assert torch.equal(y, want), i


def test_refusals_on_the_cpu():
    c, s = torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        tokens.matmul_tokens(c, s, c, s)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        tokens.linear_tokens(torch.zeros(4, 16), c, s)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        tokens.matmul_tokens(c, s, c, s, dtype=torch.int8)


@pytest.mark.gpu
def test_refusals():
    c, s = torch.zeros(4, 16, dtype=torch.int8, device=DEV), torch.zeros(4, device=DEV)
    good = (c, s, c, s)
    for i, bad, text in ((0, c.float(), "type of codes"), (1, s[:3], "one value for each row"), (1, s.double(), "type of scale"),
                         (2, c[:, :15], "features"), (2, c.view(2, 2, 16), "dimension"), (2, c.cpu(), "CUDA"), (3, s[:2], "one value for each row"),
                         (2, c.to(torch.uint8), "type of weight_codes"), (3, s.cpu(), "same device")):
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError, match=text):
            tokens.matmul_tokens(*args)
    for bias in (s[:3], s.cpu(), s.to(torch.int32)):
        with pytest.raises(RuntimeError, match="bias"):
            tokens.matmul_tokens(*good, bias=bias)
    wide = torch.zeros(1, 131072, dtype=torch.int8, device=DEV)
    with pytest.raises(RuntimeError, match="131071"):
        tokens.matmul_tokens(wide, s[:1], wide, s[:1])


def test_c_abi_refuses_bad_sizes(lib):
    f = lib.actnn_tokens_matmul
    assert f(None, 16, None, None, 16, None, None, None, 0, 16, 4, 0, None, 0, None) == 0
    assert f(None, 16, None, None, 16, None, None, None, 4, 16, 0, 0, None, 0, None) == 0
    assert f(None, 16, None, None, 16, None, None, None, 4, 16, 4, 0, None, 0, None) == -1       # null pointers
    assert f(None, 16, None, None, 16, None, None, None, 4, 17, 4, 0, None, 0, None) == -1       # rows shorter than K
    assert f(None, 24, None, None, 16, None, None, None, 4, 16, 4, 0, None, 0, None) == -1       # no multiple of 16
    assert f(None, 1 << 23, None, None, 16, None, None, None, 4, 16, 4, 0, None, 0, None) == -1  # stride
    assert f(16, 16, 16, 16, 16, 16, None, 16, 4, 16, 1 << 26, 0, None, 0, None) == -1           # more blocks than a launch takes
    assert f(16, 16, 16, 16, 16, 16, None, 16, 0x7fffff00, 16, 4, 0, None, 0, None) == -1
    assert f(None, 131072, None, None, 131072, None, None, None, 4, 131072, 4, 0, None, 0, None) == -1
    assert f(None, 16, None, None, 16, None, None, None, 4, 16, 4, 9, None, 0, None) == -2
    assert f(8, 16, 16, 16, 16, 16, None, 16, 4, 16, 4, 0, None, 0, None) == -4
    assert lib.actnn_tokens_matmul_workspace_bytes(70, 8192, 64) > 0
    few = lib.actnn_tokens_linear_few
    assert few(None, 16, None, 16, None, None, None, 0, 16, 4, 0, None) == 0
    assert few(None, 16, None, 16, None, None, None, 5, 16, 4, 0, None) == -1                    # more tokens than it takes
    assert few(None, 18, None, 32, None, None, None, 1, 18, 4, 0, None) == -1                    # no whole vectors
    assert few(16, 16, 16, 16, 16, None, 16, 1, 16, 1 << 26, 0, None) == -1
    assert few(None, 16400, None, 16400, None, None, None, 1, 16400, 4, 0, None) == -1
    assert few(None, 16, None, 16, None, None, None, 1, 16, 4, 7, None) == -2
    assert few(8, 16, 16, 16, 16, None, 16, 1, 16, 4, 0, None) == -4
    assert lib.actnn_tokens_matmul_workspace_bytes(8192, 4096, 4096) == 0
    assert lib.actnn_tokens_matmul_workspace_bytes(0, 4096, 4096) == 0
