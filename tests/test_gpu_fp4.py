"""4-bit floating point on the GPU: the quantiser byte for byte against the 64-bit oracle, the block-scaled GEMM
exactly where its sums are exact and within a bound that is counted out elsewhere.

Bound of the GEMM: with S = sum_k |x_q w_q| (no partial sum exceeds it), the tensor core adds at least 32 products
at a time, so at most K / 32 additions in fp32, each off by at most 2^-23 of S (a truncation), then up to three
roundings of the row scales and the bias (2^-24 each of at most S + |bias|); the result is rounded to the output type,
half a step of it: eps / 2 of |y| plus what came before, and at least half the type's least denormal (2^-25 for fp16).
"""
import pytest
import torch

from oracle import fp4_oracle as O4

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a B200")]

DEV = "cuda"
SCHEMES = ["mxfp4", "nvfp4"]
DTYPES = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows(M, K, dtype, seed):
    """Rows of very different size, with zeros, ties and an all-zero row."""
    g = gen(seed)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-12, 12, (M, 1), generator=g).float())
    x = x * torch.exp2(torch.randint(-8, 1, (M, K), generator=g).float())
    x[torch.rand(M, K, generator=g) < 0.1] = 0
    if M > 1:
        x[M // 2] = 0
    return x.to(dtype)


def check_quant(x, scheme):
    import fni8
    from fni8.quant import fp4

    qt = fni8.quantize_fp4(x.to(DEV), scheme)
    codes, sf, row = O4.quantize(x, scheme)
    M, K = x.shape
    assert qt.scheme == scheme and qt.cols == K and qt.group_size == fp4.BLOCK[scheme]
    assert torch.equal(fp4.scale_rows(qt.scale.cpu(), M, sf.shape[1]), sf)
    tiles = fp4.scale_tiles(sf)
    assert torch.equal(qt.scale.cpu(), tiles)  # zeros behind the rows and columns
    if row is None:
        assert qt.row_scale is None
    else:
        assert torch.equal(qt.row_scale.cpu(), row)
    bad = (sf == (0xFF if scheme == "mxfp4" else 0x7F)).repeat_interleave(fp4.BLOCK[scheme], 1)
    got = O4.unpack(qt.data.cpu())
    assert torch.equal(got[~bad], codes[~bad])
    return qt, codes, sf, row


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 4096), (2, 15), (3, 31), (5, 32), (7, 33), (129, 64), (4, 100), (128, 1023),
                                 (3, 1024), (6, 1026), (2, 2056), (1, 4097), (3, 5000), (2, 8192), (2, 8194), (1, 16500)])
def test_quantize_is_the_oracle(scheme, dtype, M, K):
    check_quant(rows(M, K, dtype, 31 * M + K), scheme)


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_every_finite_value(scheme, dtype):
    """Every finite 16-bit pattern, four to a block beside a larger one of several sizes (ties, denormals, saturation)."""
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16)
    v = bits.view(dtype)
    v = v[torch.isfinite(v.float())]
    v = torch.cat((v, torch.zeros((-v.numel()) % 1024, dtype=dtype))).view(-1, 4, 1).expand(-1, 4, 8).reshape(-1, 32)
    x = v.reshape(-1, 128).clone()
    scale = torch.tensor([1.0, 1.5, 2.0, 3.0, 5.0, 7.0, 11.0, 13.0])
    for i in range(4):  # one neighbour per block, a few times as large
        x[:, 32 * i + 7] = (x[:, 32 * i].float() * scale[torch.arange(x.shape[0]) % 8]).clamp(
            -torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)
    check_quant(x, scheme)


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties(scheme, dtype):
    """Blocks whose values sit on the borders between codes, for every e4m3 significand of the scale."""
    g = gen(5)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1.5, 6.0, -0.25, -0.75, -1.25, -2.5, -5.0, 6.0])
    blocks = []
    for sig in range(8, 16):
        for e in range(-6, 4):
            blocks.append(mids[torch.randperm(16, generator=g)] * (sig / 8) * 2.0 ** e)
    x = torch.stack(blocks).view(-1, 32).to(dtype)
    check_quant(x, scheme)


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_blocks_are_nan_alone(scheme, dtype):
    import fni8

    x = rows(4, 160, dtype, 3)
    x[0, 5] = float("inf")
    x[1, 40] = float("-inf")
    x[3, 159] = float("nan")
    qt, codes, sf, row = check_quant(x, scheme)
    g = qt.group_size
    v = fni8.dequantize_fp4(qt, torch.float32).cpu()
    want = torch.zeros(4, 160, dtype=torch.bool)
    want[0, 5 // g * g:5 // g * g + g] = True
    want[1, 40 // g * g:40 // g * g + g] = True
    want[3, 159 // g * g:159 // g * g + g] = True
    assert torch.equal(torch.isnan(v), want)
    w = fni8.quantize_fp4(rows(40, 160, dtype, 4).to(DEV), scheme)
    for m in (x, torch.cat((x, rows(300, 160, dtype, 8)))):  # both GEMM kernels
        y = fni8.linear(m.to(DEV), w).cpu()
        assert torch.equal(torch.isnan(y).all(1), want.any(1) if m is x else torch.cat((want.any(1), torch.zeros(300, dtype=torch.bool))))
        assert not torch.isnan(y[2]).any()


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 40), (130, 96), (2, 4099)])
def test_dequantize_is_the_oracle(scheme, M, K):
    import fni8

    qt, codes, sf, row = check_quant(rows(M, K, torch.bfloat16, K), scheme)
    if row is not None:  # any fp32 row scale
        qt.row_scale = (row * (0.5 + torch.rand(M, generator=gen(9)))).to(DEV)
        row = qt.row_scale.cpu()
    want = O4.values(codes, sf, row, scheme)[:, :K]
    assert torch.equal(fni8.dequantize_fp4(qt, torch.float32).cpu(), want.float())
    for dt in DTYPES:
        assert torch.equal(fni8.dequantize_fp4(qt, dt).cpu(), want.float().to(dt))


def random_qt(N, K, scheme, seed, exact):
    """A weight with any codes. exact: scales of a few powers of two, row scales of powers of two, so that every sum of
    products is a multiple of 2^-8 below 2^16 and fp32 holds it exactly."""
    import fni8
    from fni8.quant import fp4

    g = gen(seed)
    Kp, b = (K + 31) // 32 * 32, fp4.BLOCK[scheme]
    codes = torch.randint(0, 16, (N, Kp), generator=g, dtype=torch.uint8)
    codes[:, K:] = 0
    n = Kp // b
    if exact:
        e = torch.randint(-1, 2, (N, n), generator=g)
        sf = (e + 127).to(torch.uint8) if scheme == "mxfp4" else torch.exp2(e.float()).to(torch.float8_e4m3fn).view(torch.uint8)
        row = torch.exp2(torch.randint(-2, 3, (N,), generator=g).float())
    else:
        sf = torch.randint(118, 128, (N, n), generator=g, dtype=torch.uint8) if scheme == "mxfp4" else \
            (0.01 + 100 * torch.rand(N, n, generator=g)).to(torch.float8_e4m3fn).view(torch.uint8)
        row = 0.001 + torch.rand(N, generator=g)
    row = row if scheme == "nvfp4" else None
    qt = fni8.QTensor(O4.pack(codes), fp4.scale_tiles(sf), scheme=scheme, group_size=b, row_scale=row, cols=K)
    return qt.to(DEV), O4.values(codes, sf, row, scheme)[:, :K]


SHAPES = [(1, 8, 32), (1, 1, 1), (2, 129, 64), (3, 200, 96), (16, 256, 256), (17, 130, 320), (33, 1030, 288), (64, 128, 4096),
          (100, 384, 1000), (128, 512, 2048), (129, 640, 512), (200, 77, 130), (256, 1024, 1024), (300, 264, 2080),
          (513, 520, 736), (1100, 2056, 544), (100, 300, 4100), (65, 128, 9000), (129, 130, 4096), (300, 1030, 6000),
          (513, 129, 4097), (120, 19000, 300), (300, 13000, 70), (1000, 4200, 328), (128, 40000, 96)]


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_exact_sums(scheme, M, N, K):
    """Operands whose sums fp32 holds: the result is the rounded sum, bit for bit."""
    import fni8

    dtype = DTYPES[(M + N) % 2]
    a, av = random_qt(M, K, scheme, M + K, True)
    w, wv = random_qt(N, K, scheme, N + K, True)
    y = fni8.linear_fp4(a, w, out_dtype=dtype).cpu()
    want = (av.to(DEV) @ wv.to(DEV).t()).cpu()
    assert torch.equal(y, want.float().to(dtype))
    assert fni8.device_status() == 0


def bound(av, wv, y, bias, dtype, K):
    S = av.abs().to(DEV) @ wv.abs().to(DEV).t()
    S = S.cpu() + (0 if bias is None else bias.double().abs())
    pre = (K / 32 + 1) * 2.0 ** -23 * S + 3 * 2.0 ** -24 * S
    return pre + torch.finfo(dtype).eps / 2 * (y.abs() + pre) + 2.0 ** -25


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("M,N,K", SHAPES + [(8, 4096, 12288), (700, 512, 12288)])
def test_gemm_within_bound(scheme, M, N, K):
    import fni8

    dtype = DTYPES[(M + N + K) % 2]
    a, av = random_qt(M, K, scheme, M, False)
    w, wv = random_qt(N, K, scheme, N, False)
    bias = torch.randn(N, generator=gen(K)).to(dtype) if M % 2 else None
    y = fni8.linear_fp4(a, w, bias=None if bias is None else bias.to(DEV), out_dtype=dtype).cpu().double()
    want = (av.to(DEV) @ wv.to(DEV).t()).cpu()
    if bias is not None:
        want = want + bias.double()
    tol = bound(av, wv, want, bias, dtype, K)
    # a value that rounds past the type's largest is an infinity of its sign, on either side of the border within tol
    top = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)
    inf = torch.isinf(y)
    assert (want.abs()[inf] + tol[inf] >= top).all() and torch.equal(y[inf].sign(), want[inf].sign())
    assert ((y - want).abs() <= tol)[~inf].all(), float((y - want)[~inf].abs().max())


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,N,K", [((1,), 6144, 4096), ((2, 5), 96, 70), ((400,), 1030, 1080), ((), 64, 64), ((0,), 64, 64)])
def test_linear_is_quantise_then_gemm(scheme, dtype, lead, N, K):
    import fni8

    g = gen(N)
    x = torch.randn(*lead, K, generator=g).to(dtype).to(DEV)
    w = fni8.quantize_fp4((0.05 * torch.randn(N, K, generator=g)).to(dtype).to(DEV), scheme)
    bias = torch.randn(N, generator=g).to(dtype).to(DEV)
    y = fni8.linear(x, w, bias=bias)
    assert y.shape == (*lead, N) and y.dtype == dtype
    if x.dim() > 1:
        assert torch.equal(y, fni8.linear_fp4(fni8.quantize_fp4(x, scheme), w, bias=bias, out_dtype=dtype))
    if x.numel():
        full = x.reshape(-1, K).double().cpu() @ fni8.dequantize_fp4(w, torch.float32).double().cpu().t() + bias.double().cpu()
        cos = torch.nn.functional.cosine_similarity(y.double().cpu().flatten(), full.flatten(), dim=0)
        assert cos > 0.98, cos


@pytest.mark.parametrize("scheme", SCHEMES)
def test_strides_and_devices(scheme):
    """Rows that are views (every second row, a column slice, an odd offset), as any other input of fni8.linear."""
    import fni8

    w = fni8.quantize_fp4(torch.randn(96, 200, generator=gen(1)).half().to(DEV), scheme)
    base = torch.randn(20, 403, generator=gen(2)).half().to(DEV)
    for v in (base[::2, :200], base[:, 3:203], base.t()[100:300, :].t()):
        assert torch.equal(fni8.linear(v, w), fni8.linear(v.clone(memory_format=torch.contiguous_format), w))
    flat = torch.randn(1 + 7 * 200, generator=gen(3)).half().to(DEV)
    odd = flat[1:].view(7, 200)  # 2-byte aligned rows
    assert torch.equal(fni8.quantize_fp4(odd, scheme).data, fni8.quantize_fp4(odd.clone(), scheme).data)


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("M", [4, 300])
def test_graph_replay_and_side_stream(scheme, M):
    import fni8

    N, K = 640, 1024
    w = fni8.quantize_fp4(torch.randn(N, K, generator=gen(1)).half().to(DEV), scheme)
    x = torch.randn(M, K, generator=gen(2)).half().to(DEV)
    fni8.linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fni8.linear(x, w)
        z = fni8.dequantize_fp4(fni8.quantize_fp4(x, scheme), torch.float16)
    for seed in (3, 4):
        x.copy_(torch.randn(M, K, generator=gen(seed)).half())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fni8.linear(x, w))
        assert torch.equal(z, fni8.dequantize_fp4(fni8.quantize_fp4(x, scheme)))
    side = torch.cuda.Stream()
    xs = [torch.randn(M, K, generator=gen(10 + i)).half().to(DEV) for i in range(4)]
    want = [fni8.linear(v, w) for v in xs]
    torch.cuda.synchronize()
    got = [None] * 4
    for i, v in enumerate(xs):  # two streams at once: no shared workspace
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            got[i] = fni8.linear(v, w)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gated_mlp_with_fp4_weights():
    """A module of the framework over such weights: norm -> GatedMLP, equal to its calls one by one."""
    import fni8
    from fni8.mlp import GatedMLP

    H, I = 512, 384
    for scheme in SCHEMES:
        gu = fni8.quantize_fp4((0.05 * torch.randn(2 * I, H, generator=gen(1))).half().to(DEV), scheme)
        dn = fni8.quantize_fp4((0.05 * torch.randn(H, I, generator=gen(2))).half().to(DEV), scheme)
        mlp = GatedMLP(gu, dn)
        for M in (3, 500):
            x = fni8.rmsnorm(torch.randn(M, H, generator=gen(M)).half().to(DEV), torch.ones(H).half().to(DEV), 1e-6)
            want = fni8.linear(fni8.act_and_mul(fni8.linear(x, gu)), dn)
            got = mlp(x)
            assert torch.equal(got, want) and torch.isfinite(got).all() and float(got.abs().max()) > 0


def test_refusals_on_the_gpu():
    import fni8

    w = fni8.quantize_fp4(torch.randn(32, 64, generator=gen(1)).half().to(DEV), "mxfp4")
    x = torch.randn(4, 64, generator=gen(2)).half().to(DEV)
    with pytest.raises(TypeError):
        fni8.quantize_fp4(x.float())
    with pytest.raises(ValueError):
        fni8.quantize_fp4(x, "int4")
    with pytest.raises(ValueError):
        fni8.linear(x[:, :60], w)
    with pytest.raises(ValueError):
        fni8.linear(x, w, bias=torch.zeros(31, device=DEV).half())
    with pytest.raises(ValueError):
        fni8.linear_fp4(fni8.quantize_fp4(x, "nvfp4"), w)
    with pytest.raises(TypeError):
        fni8.linear_fp4(fni8.quantize_fp4(x), w, out_dtype=torch.float32)
    with pytest.raises(TypeError):
        fni8.dequantize_fp4(w, torch.int8)
    with pytest.raises(RuntimeError):
        fni8.linear(x, w.to("cpu"))


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 128, 8), (1, 129, 256), (3, 6144, 4096), (16, 96, 1000), (7, 4096, 12288),
                                   (16, 20000, 520), (5, 40000, 2048), (9, 300, 8200), (2, 130, 16384), (17, 200, 4096)])
def test_linear_in_one_kernel(scheme, dtype, M, N, K):
    """Up to 16 rows linear quantises them in the GEMM: the result of the two calls bit for bit, also with rows of
    very different size, an all-zero row, and from misaligned rows (which take the two kernels)."""
    import fni8

    x = rows(M, K, dtype, M + K).to(DEV)
    w, _ = random_qt(N, K, scheme, N, False)
    bias = torch.randn(N, generator=gen(3)).to(dtype).to(DEV)
    want = fni8.linear_fp4(fni8.quantize_fp4(x, scheme), w, bias=bias, out_dtype=dtype)
    for _ in range(2):
        assert torch.equal(fni8.linear(x, w, bias=bias), want)
    flat = torch.empty(M * K + 1, dtype=dtype, device=DEV)
    flat[1:] = x.reshape(-1)
    assert torch.equal(fni8.linear(flat[1:].view(M, K), w, bias=bias), want)
    assert fni8.device_status() == 0


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("M", [1, 40, 300])
def test_weights_quantised_right_before(scheme, M):
    """linear directly behind the kernel that writes its weights, on the memory that the last weights had."""
    import fni8

    N, K = 12288, 4096
    x = torch.randn(M, K, generator=gen(1)).half().to(DEV)
    ws = [0.05 * torch.randn(N, K, device=DEV, dtype=torch.float16) * (i + 1) for i in range(4)]
    torch.cuda.synchronize()
    got = []
    for w in ws:
        q = fni8.quantize_fp4(w, scheme)
        got.append(fni8.linear(x, q))
        del q
    for w, y in zip(ws, got):
        q = fni8.quantize_fp4(w, scheme)
        torch.cuda.synchronize()
        assert torch.equal(fni8.linear(x, q), y)


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("lead", [(), (2, 3), (0,), (4, 0)])
def test_leading_dims(scheme, lead):
    """Any leading dims, none at all among them: the values, codes and product of the flattened rows."""
    import fni8

    K, N = 70, 48
    x = torch.randn(*lead, K, generator=gen(1)).half().to(DEV)
    w = fni8.quantize_fp4(torch.randn(N, K, generator=gen(2)).half().to(DEV), scheme)
    q, flat = fni8.quantize_fp4(x, scheme), fni8.quantize_fp4(x.reshape(-1, K), scheme)
    assert fni8.dequantize_fp4(q).shape == x.shape
    assert torch.equal(fni8.dequantize_fp4(q).reshape(-1, K), fni8.dequantize_fp4(flat))
    for y in (fni8.linear(x, w), fni8.linear_fp4(q, w)):
        assert y.shape == (*lead, N)
        assert torch.equal(y.reshape(-1, N), fni8.linear_fp4(flat, w))


@pytest.mark.parametrize("scheme", SCHEMES)
def test_shards_give_the_columns(scheme):
    import fni8
    from fni8.parallel import shard_rows

    x = torch.randn(40, 320, generator=gen(1)).half().to(DEV)
    w = fni8.quantize_fp4(torch.randn(300, 320, generator=gen(2)).half().to(DEV), scheme)
    y = torch.cat([fni8.linear(x, shard_rows(w, 3, r)) for r in range(3)], dim=1)
    assert torch.equal(y, fni8.linear(x, w))
