"""4-bit floating point on the host: the oracle against hand-worked values, the tile order of the scales, the
container, and every refusal of the C ABI and the Python layer (no GPU)."""
import ctypes

import pytest
import torch

from oracle import fp4_oracle as O4


def test_oracle_mxfp4_hand_worked():
    x = torch.zeros(1, 32, dtype=torch.float16)
    # max 7 -> floor(log2 7) = 2 -> scale 2^0: codes are the values themselves
    x[0, :9] = torch.tensor([7.0, 6.0, -5.0, 3.5, 2.5, 0.25, 0.75, -0.5, 1.25])
    codes, sf, row = O4.quantize(x, "mxfp4")
    assert row is None and sf.tolist() == [[127]]
    got = O4.values(codes, sf, row, "mxfp4")[0, :9].tolist()
    # 7 saturates; 5 -> 4, 3.5 -> 4, 2.5 -> 2, 0.25 -> 0, 0.75 -> 1, 1.25 -> 1 (ties to the even code)
    assert got == [6, 6, -4, 4, 2, 0, 1, -0.5, 1]


def test_oracle_nvfp4_hand_worked():
    x = torch.zeros(2, 32, dtype=torch.float32)
    x[0, 0], x[0, 16] = 2688.0, 6.0  # row scale 1, block scales 448 and 1
    x[0, 17] = -2.5
    x[1, 0] = 2689.0  # just above: row scale 2
    codes, sf, row = O4.quantize(x, "nvfp4")
    assert row.tolist() == [1.0, 2.0]
    assert sf.view(torch.float8_e4m3fn).float()[0].tolist() == [448.0, 1.0]
    v = O4.values(codes, sf, row, "nvfp4")
    assert v[0, 0] == 2688 and v[0, 16] == 6 and v[0, 17] == -2


def test_scale_tiles_round_trip_and_order():
    from fni8.quant import fp4

    for N, S in ((1, 1), (128, 4), (130, 9), (257, 5)):
        rows = torch.randint(0, 256, (N, S), dtype=torch.uint8, generator=torch.Generator().manual_seed(N))
        t = fp4.scale_tiles(rows)
        assert t.shape == ((N + 127) // 128, (S + 3) // 4, 512)
        assert torch.equal(fp4.scale_rows(t, N, S), rows)
        for r in {0, N // 2, N - 1}:
            for s in {0, S // 2, S - 1}:
                assert t[r // 128, s // 4, r % 32 * 16 + r % 128 // 32 * 4 + s % 4] == rows[r, s]
        assert int(t.long().sum()) == int(rows.long().sum())  # zeros elsewhere
    with pytest.raises(ValueError):
        fp4.scale_tiles(torch.zeros(3, 4))
    with pytest.raises(ValueError):
        fp4.scale_rows(torch.zeros(1, 1, 512, dtype=torch.uint8), 129, 4)


@pytest.mark.parametrize("scheme", ["mxfp4", "nvfp4"])
def test_container_round_trip(tmp_path, scheme):
    import fni8
    from fni8.quant import fp4

    codes, sf, row = O4.quantize(torch.randn(130, 70, generator=torch.Generator().manual_seed(1)).half(), scheme)
    qt = fni8.QTensor(O4.pack(codes), fp4.scale_tiles(sf), scheme=scheme, group_size=fp4.BLOCK[scheme], row_scale=row,
                      cols=70)
    path = str(tmp_path / "w.fni8")
    fni8.save_fni8(path, {"w": qt})
    with fni8.FQReader(path) as r:
        assert r.header["quant"] == scheme
        back = r.load_many(["w"])["w"]
    assert torch.equal(back.data, qt.data) and torch.equal(back.scale, qt.scale)
    assert back.scheme == scheme and back.cols == 70 and back.group_size == qt.group_size
    assert (back.row_scale is None) if row is None else torch.equal(back.row_scale, row)


def test_c_abi_refusals():
    from fni8 import _native as n

    L = n.lib()
    p, bad = 4096, 4096 + 8  # addresses that are only looked at: every call is refused on the host

    def quant(x=p, dt=n.F16, fmt=n.MXFP4, M=4, K=64, q=p, sf=p, rs=p):
        return L.fni8_quantize_rows_fp4(x, dt, fmt, M, K, q, sf, rs, None)

    assert quant(dt=n.F32) == n.ERR_INVALID
    assert quant(fmt=2) == n.ERR_INVALID
    assert quant(M=-1) == n.ERR_INVALID and quant(K=0) == n.ERR_INVALID
    assert quant(M=1 << 31) == n.ERR_UNSUPPORTED and quant(K=1 << 31) == n.ERR_UNSUPPORTED
    assert quant(x=None) == n.ERR_INVALID and quant(q=None) == n.ERR_INVALID and quant(sf=None) == n.ERR_INVALID
    assert quant(fmt=n.NVFP4, rs=None) == n.ERR_INVALID
    assert quant(x=p + 1) == n.ERR_ALIGN and quant(q=bad) == n.ERR_ALIGN and quant(sf=bad) == n.ERR_ALIGN
    assert quant(M=0, x=None) == n.OK

    def deq(q=p, sf=p, rs=p, fmt=n.MXFP4, M=4, K=64, out=p, dt=n.F16):
        return L.fni8_dequantize_rows_fp4(q, sf, rs, fmt, M, K, out, dt, None)

    assert deq(dt=n.I8) == n.ERR_INVALID and deq(fmt=-1) == n.ERR_INVALID and deq(K=0) == n.ERR_INVALID
    assert deq(q=None) == n.ERR_INVALID and deq(out=None) == n.ERR_INVALID
    assert deq(fmt=n.NVFP4, rs=None) == n.ERR_INVALID and deq(q=p + 2) == n.ERR_ALIGN
    assert deq(M=0, q=None) == n.OK

    def gemm(a=p, asf=p, ars=p, w=p, wsf=p, wrs=p, bias=None, out=p, dt=n.F16, fmt=n.NVFP4, M=4, N=8, K=64):
        return L.fni8_gemm_fp4(a, asf, ars, w, wsf, wrs, bias, out, dt, fmt, M, N, K, None)

    assert gemm(dt=n.F32) == n.ERR_INVALID and gemm(fmt=7) == n.ERR_INVALID
    assert gemm(M=-1) == n.ERR_INVALID and gemm(N=0) == n.ERR_INVALID and gemm(K=0) == n.ERR_INVALID
    assert gemm(M=1 << 31) == n.ERR_UNSUPPORTED and gemm(N=1 << 30, K=1 << 16) == n.ERR_UNSUPPORTED
    for name in ("a", "asf", "ars", "w", "wsf", "wrs", "out"):
        assert gemm(**{name: None}) == n.ERR_INVALID, name
    for name in ("a", "asf", "w", "wsf"):
        assert gemm(**{name: bad}) == n.ERR_ALIGN, name
    assert gemm(out=p + 1) == n.ERR_ALIGN and gemm(bias=p + 1) == n.ERR_ALIGN
    assert gemm(M=0, a=None) == n.OK

    def linear(x=p, dt=n.BF16, fmt=n.NVFP4, M=40, N=8, K=64, w=p, scratch=p, sb=1 << 20):
        return L.fni8_linear_fp4(x, dt, w, p, p, None, p, fmt, M, N, K, scratch, sb, None)

    assert linear(x=None) == n.ERR_INVALID and linear(w=None) == n.ERR_INVALID and linear(N=-3) == n.ERR_INVALID
    assert linear(dt=n.I32) == n.ERR_INVALID and linear(fmt=3) == n.ERR_INVALID
    need = L.fni8_linear_fp4_scratch_bytes(n.NVFP4, 40, 8, 64)
    assert need == 512 + 40 * 32 + 40 * 4
    assert linear(scratch=None) == n.ERR_WORKSPACE and linear(sb=need - 1) == n.ERR_WORKSPACE
    assert linear(scratch=bad) == n.ERR_ALIGN and linear(x=p + 1) == n.ERR_ALIGN
    # one kernel, for what its threads hold in registers
    assert L.fni8_linear_fp4_scratch_bytes(n.MXFP4, 16, 8, 64) == 0 and L.fni8_linear_fp4_scratch_bytes(n.NVFP4, 8, 8, 64) == 0
    assert L.fni8_linear_fp4_scratch_bytes(n.NVFP4, 16, 8, 64) > 0
    assert linear(M=8, x=bad, scratch=None, sb=0) == n.ERR_ALIGN
    assert L.fni8_linear_fp4_scratch_bytes(n.NVFP4, 16, 8, 63) > 0 and linear(M=16, K=63, sb=0) == n.ERR_WORKSPACE
    assert L.fni8_linear_fp4_scratch_bytes(9, 16, 8, 64) == 0 and L.fni8_linear_fp4_scratch_bytes(0, 0, 8, 64) == 0
    assert linear(M=0, x=None) == n.OK
    assert L.fni8_fp4_scale_bytes(n.MXFP4, 130, 129) == 2 * 2 * 512
    assert L.fni8_fp4_scale_bytes(n.NVFP4, 1, 64) == 512
    assert L.fni8_fp4_scale_bytes(5, 1, 64) == 0 and L.fni8_fp4_scale_bytes(n.MXFP4, 0, 64) == 0
    assert isinstance(L.fni8_last_error_message(), bytes) and ctypes.sizeof(ctypes.c_void_p) == 8


def test_python_refusals():
    import fni8
    from fni8.quant import fp4
    from fni8.ops import _fp4_shape

    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        fni8.quantize_fp4(x)  # CPU tensor
    codes, sf, row = O4.quantize(x, "nvfp4")
    parts = dict(scheme="nvfp4", group_size=16, row_scale=row, cols=64)
    ok = fni8.QTensor(O4.pack(codes), fp4.scale_tiles(sf), **parts)
    assert _fp4_shape(ok, "t") == (4, 64)
    for change in (dict(group_size=32), dict(row_scale=None), dict(row_scale=row[:3]), dict(row_scale=row.double()),
                   dict(cols=65), dict(cols=32), dict(scheme="mxfp4"), dict(scheme="per_row_i8")):
        with pytest.raises(ValueError):
            _fp4_shape(fni8.QTensor(ok.data, ok.scale, **{**parts, **change}), "t")
    with pytest.raises(ValueError):
        _fp4_shape(fni8.QTensor(ok.data, ok.scale[:, :0], **parts), "t")
    with pytest.raises(ValueError):
        _fp4_shape(fni8.QTensor(ok.data.view(torch.int8), ok.scale, **parts), "t")
    with pytest.raises(ValueError):
        _fp4_shape(fni8.QTensor(ok.data.t().contiguous().t(), ok.scale, **parts), "t")
    with pytest.raises(RuntimeError):
        fni8.dequantize_fp4(ok)
    with pytest.raises(RuntimeError):
        fni8.linear_fp4(ok, ok)
    with pytest.raises(RuntimeError):
        fni8.linear(x, ok)


@pytest.mark.parametrize("scheme", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("N,world", [(256, 2), (260, 4), (9, 3)])
def test_row_shards(scheme, N, world):
    """An output-channel shard is the rows' own codes, scales and row scales, whatever tile they were in."""
    import fni8
    from fni8.parallel import shard_rows
    from fni8.quant import fp4

    codes, sf, row = O4.quantize(torch.randn(N, 200, generator=torch.Generator().manual_seed(N)).half(), scheme)
    qt = fni8.QTensor(O4.pack(codes), fp4.scale_tiles(sf), scheme=scheme, group_size=fp4.BLOCK[scheme], row_scale=row,
                      cols=200)
    n = N // world
    for r in range(world):
        s = shard_rows(qt, world, r)
        own = slice(r * n, (r + 1) * n)
        assert s.scheme == scheme and s.group_size == qt.group_size and s.cols == 200
        assert torch.equal(s.data, qt.data[own])
        assert torch.equal(fp4.scale_rows(s.scale, n, sf.shape[1]), sf[own])
        assert torch.equal(s.scale, fp4.scale_tiles(sf[own]))
        assert s.row_scale is None if row is None else torch.equal(s.row_scale, row[own])
    with pytest.raises(ValueError):
        shard_rows(qt, 7, 0)
