"""8-bit tokens against their definition in 64 bits: codes exactly, values to the roundings they are made of."""
import pytest
import torch

from actnn_amd.cpp_extension import tokens
from oracle import tokens as oracle

DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(M, K, dtype, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=gen) * torch.exp(spread * torch.randn(M, 1, generator=gen))
    return x.to(dtype)


def check_codes(x, codes, scale, where=""):
    q, s = oracle.codes(x)
    assert codes.dtype == torch.int8 and codes.shape == x.shape and scale.shape == x.shape[:-1]
    assert torch.equal(codes.cpu().double(), q), where
    # one rounding of top / 127 to 32 bits; at most the largest scale whose 127-fold is finite (fp32's largest value over 127
    # rounds up to 0x1.020408p121, and 127 times that is 0x1.000000p128 rounded: an infinity)
    s = s.squeeze(-1).clamp(max=float.fromhex("0x1.020406p121"))
    got = scale.cpu().double()
    assert ((got - s).abs() <= 2.0 ** -24 * s.abs()).logical_or(torch.isnan(s) & torch.isnan(got)).all(), where


# rows of a wave with 1, 2 and 4 vectors, of a block with 1 to 8, read twice; odd ones; single tokens; tensors below 16 bytes
SHAPES = [(1, 1), (1, 3), (2, 3), (3, 1), (1, 7), (1, 17), (5, 16), (7, 33), (130, 64), (9, 257), (1025, 130), (1030, 1001),
          (1024, 2048), (3, 2040), (2, 4096), (5, 4099), (1, 8192), (2, 10000), (1, 16384), (3, 16390), (1, 70001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", SHAPES)
def test_codes_are_exactly_the_definition(M, K, dtype):
    print(f"[tokens] {M}x{K} {dtype}", flush=True)
    x = make(M, K, dtype, M + K)
    codes, scale = tokens.quantize_tokens(x.to(DEV))
    assert M < 2 or codes.stride(0) == (K + 15) // 16 * 16
    check_codes(x, codes, scale)
    for out in DTYPES:
        v = tokens.dequantize_tokens(codes, scale, out)
        exact = codes.cpu().double() * scale.cpu().double()[:, None]
        assert v.dtype == out and v.shape == x.shape
        bound = HALF_STEP[out] * exact.abs() + (2.0 ** -25 if out == torch.float16 else 0.0)   # + half of fp16's smallest
        # (the product is rounded to 32 bits on its way to 16)
        assert ((v.cpu().double() - exact).abs() <= bound + 2.0 ** -24 * exact.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_half_is_rounded_up(dtype):
    # all significands of a type against tops whose halves they meet: 127 x / top = q + 1/2 for odd multiples of top / 254,
    # and the neighbours of those values on both sides
    rows = []
    for top in (127.0, 254.0, 381.0, 1016.0, 127.0 * 15, 1.0, 3.0, 2.0 ** -14 * 127):
        q = torch.arange(0, 127, dtype=torch.float64)
        x = ((q + 0.5) * top / 127.0).to(dtype)
        step = torch.nextafter(x, torch.full_like(x, float("inf"))), torch.nextafter(x, torch.zeros_like(x))
        row = torch.cat([x, *step, torch.tensor([top], dtype=dtype)])
        rows.append(torch.cat([row, -row]))
    x = torch.stack(rows)
    codes, scale = tokens.quantize_tokens(x.to(DEV))
    check_codes(x, codes, scale)
    assert (codes.cpu() == 127).any(dim=1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_16_bit_value_against_many_tops(dtype):
    gen = torch.Generator().manual_seed(5)
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    every = every[torch.isfinite(every)]
    tops = every[torch.randint(0, every.numel(), (64,), generator=gen)].abs()
    tops = torch.cat([tops, torch.tensor([1.0, 127.0, 1.9921875, 65504.0]).to(dtype)])
    rows = torch.where(every[None].abs() <= tops[:, None], every[None], torch.zeros((), dtype=dtype))
    rows[:, 0] = tops
    codes, scale = tokens.quantize_tokens(rows.to(DEV))
    check_codes(rows, codes, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [5, 64, 300, 5000, 20000])
def test_rows_of_zeros_tiny_values_nan_and_infinity(K, dtype):
    x = make(8, K, torch.float32, K).to(dtype)
    x[1] = 0
    x[2] = -0.0
    x[3, K // 2] = float("nan")
    x[4, K - 1] = float("inf")
    x[5, 0] = float("-inf")
    x[6] = 0
    x[6, K // 3] = torch.finfo(dtype).smallest_normal if dtype != torch.float16 else 0.0   # below 2^-100: counts as zero
    x[7, 1] = torch.finfo(dtype).max
    codes, scale = tokens.quantize_tokens(x.to(DEV))
    check_codes(x, codes, scale)
    v = tokens.dequantize_tokens(codes, scale, dtype).cpu()
    assert torch.isnan(v[3:6]).all() and (v[[1, 2, 6]] == 0).all() and torch.isfinite(v[[0, 7]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_offsets_and_leading_dimensions(dtype):
    base = make(40, 1024, dtype, 3).to(DEV)
    for x in (base[:1, :3].expand(1000, 3), base[:1, 5:6].expand(70, 1), base[:, 3:700], base[::3, :513], base[5:6, 1:], base.t()[:77], base[:1].expand(9, 1024), base.view(4, 10, 1024)[:, 2:5, 8:80],
              base.view(2, 2, 10, 1024)[1:], base[0], base[:, 100:101], base[3:3]):
        codes, scale = tokens.quantize_tokens(x)
        check_codes(x, codes, scale)
        again = tokens.dequantize_tokens(codes, scale, dtype)
        for other in (codes.contiguous(), codes.clone().t().contiguous().t() if x.dim() == 2 else codes.clone()):   # laid out otherwise
            assert torch.equal(tokens.dequantize_tokens(other, scale, dtype), again)


@pytest.mark.gpu
def test_nothing_behind_the_rows_is_written():
    # the last row's padding ends the allocation of the codes
    from actnn_amd import _lib
    lib = _lib.load()
    x = make(6, 37, torch.bfloat16, 1).to(DEV)
    room = torch.full((6 * 48 + 64,), 77, dtype=torch.int8, device=DEV)
    scale = torch.empty(8, device=DEV).fill_(7.0)
    assert lib.actnn_tokens_quantize(x.data_ptr(), 37, room.data_ptr(), 48, scale.data_ptr(), 6, 37, 2,
                                     torch.cuda.current_stream().cuda_stream) == 0
    assert (room[6 * 48:] == 77).all() and (scale[6:] == 7).all()
    assert (room[:288].view(6, 48)[:, 37:] == 0).all()
    out = torch.full((6 * 37 + 9,), 5.0, device=DEV, dtype=torch.float16)
    assert lib.actnn_tokens_dequantize(room.data_ptr(), 48, scale.data_ptr(), out.data_ptr(), 6, 37, 1,
                                       torch.cuda.current_stream().cuda_stream) == 0
    assert (out[6 * 37:] == 5).all()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    # 2.4e9 values: the last rows are what they are by themselves, through every operator that walks over tokens
    M, K, O = 300_000, 8192, 24
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=DEV)
    tail = make(300, K, torch.bfloat16, 9).to(DEV)
    x[-300:] = tail
    codes, scale = tokens.quantize_tokens(x)
    c, s = tokens.quantize_tokens(tail)
    assert torch.equal(codes[-300:], c) and torch.equal(scale[-300:], s) and not scale[:-300].any() and not codes[M // 2].any()
    del x
    assert torch.equal(tokens.dequantize_tokens(codes, scale, torch.bfloat16)[-300:], tokens.dequantize_tokens(c, s, torch.bfloat16))
    wcodes, wscale = tokens.quantize_tokens(torch.randn(O, K, device=DEV))
    y = tokens.matmul_tokens(codes, scale, wcodes, wscale)
    assert torch.equal(y[-300:], tokens.matmul_tokens(c, s, wcodes, wscale)) and not y[:-300].any()
    g = torch.zeros(M, O, dtype=torch.bfloat16, device=DEV)
    g[-300:] = torch.randn(300, O, device=DEV)
    gw = tokens.linear_tokens_grad_weight(g, codes, scale, torch.float32)
    values = (c.float() * s[:, None]).bfloat16().double()
    exact, size = g[-300:].double().t() @ values, g[-300:].double().abs().t() @ values.abs()
    assert ((gw.double() - exact).abs() <= 2.0 ** -23 * 302 * size).all()


@pytest.mark.gpu
def test_more_rows_than_a_row_of_blocks():
    # (four rows to a block, and one)
    for M, K in ((2 ** 26 + 5, 8), (2 ** 20 + 3, 2056)):
        print(f"[tokens] {M}x{K}", flush=True)
        x = make(1, K, torch.float16, K).to(DEV)
        codes, scale = tokens.quantize_tokens(x.expand(M, K))
        c, s = tokens.quantize_tokens(x)
        assert (codes == c).all() and (scale == s).all()
        assert (tokens.dequantize_tokens(codes, scale, torch.float16) == tokens.dequantize_tokens(c, s, torch.float16)).all()


@pytest.mark.gpu
def test_tokens_on_another_stream():
    x = make(512, 1024, torch.bfloat16, 2).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        codes, scale = tokens.quantize_tokens(x)
        v = tokens.dequantize_tokens(codes, scale, torch.bfloat16)
    torch.cuda.current_stream().wait_stream(side)
    check_codes(x, codes, scale)
    assert torch.equal(v, tokens.dequantize_tokens(*tokens.quantize_tokens(x), torch.bfloat16))


def test_refusals():
    x = torch.zeros(4, 16)
    for call in (lambda: tokens.quantize_tokens(x), lambda: tokens.dequantize_tokens(x.to(torch.int8), x[:, 0])):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        tokens.dequantize_tokens(x.to(torch.int8), x[:, 0], torch.float64)
    with pytest.raises(TypeError):
        tokens.quantize_tokens([1.0, 2.0])


@pytest.mark.gpu
def test_refusals_of_gpu_tensors():
    x = torch.zeros(4, 16, device=DEV)
    for bad in (x.double(), x.to(torch.int32)):
        with pytest.raises(RuntimeError, match="type of data"):
            tokens.quantize_tokens(bad)
    for bad in (x[0, 0], x[:, :0]):
        with pytest.raises(RuntimeError, match="at least one"):
            tokens.quantize_tokens(bad)
    codes, scale = tokens.quantize_tokens(x)
    for c, s in ((x, scale), (codes, scale.double()), (codes, scale[:3]), (codes, scale.cpu())):
        with pytest.raises(RuntimeError):
            tokens.dequantize_tokens(c, s)


def test_c_abi_refuses_bad_sizes(lib):
    q, d = lib.actnn_tokens_quantize, lib.actnn_tokens_dequantize
    assert q(None, 16, None, 16, None, -1, 16, 0, None) == -1
    assert q(None, 16, None, 16, None, 1, 0, 0, None) == -1
    assert q(None, 16, None, 24, None, 1, 16, 0, None) == -1          # rows of codes at multiples of 16
    assert q(None, 16, None, 16, None, 1, 17, 0, None) == -1          # shorter than the row
    assert q(None, 16, None, 16, None, 1, 16, 3, None) == -2
    assert q(None, 16, None, 16, None, 0, 16, 0, None) == 0
    assert q(None, 16, None, 16, None, 1, 16, 0, None) == -1          # null pointers
    assert q(16, 16, 8, 16, 16, 1, 16, 0, None) == -4
    assert d(None, 16, None, None, 0, 16, 0, None) == 0
    assert d(None, 8, None, None, 1, 8, 0, None) == -1
    assert d(16, 16, 16, 2, 1, 16, 0, None) == -4
