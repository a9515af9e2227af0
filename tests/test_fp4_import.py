"""4-bit floating point weights as a checkpoint holds them (codes [N, K / 2], scale bytes [N, K / block]) into the
kernels' layout, for any K that the format allows."""
import pytest
import torch

DEV = "cuda"
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
SIZES = [("nvfp4", 16), ("nvfp4", 48), ("nvfp4", 1040), ("nvfp4", 1024), ("mxfp4", 32), ("mxfp4", 96), ("mxfp4", 1056)]
E4M3 = {0.5: 0x30, 1.0: 0x38, 2.0: 0x40}


def checkpoint(N, K, scheme, seed):
    """(packed codes, scale bytes, the weight's values in 64 bits)."""
    g = torch.Generator().manual_seed(seed)
    block = 16 if scheme == "nvfp4" else 32
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    scale = torch.tensor([0.5, 1.0, 2.0])[torch.randint(0, 3, (N, K // block), generator=g)]
    if scheme == "nvfp4":
        raw = torch.zeros_like(scale, dtype=torch.uint8)
        for v, b in E4M3.items():
            raw[scale == v] = b
    else:
        raw = (torch.log2(scale) + 127).to(torch.uint8)
    values = GRID[codes.long()] * scale.double().repeat_interleave(block, 1)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), raw, values


def qtensor(packed, raw, scheme, K):
    import fni8
    from fni8.quant import fp4

    rs = torch.ones(packed.shape[0]) if scheme == "nvfp4" else None
    return fni8.QTensor(fp4.pad_codes(packed, K), fp4.scale_tiles(raw), scheme=scheme, row_scale=rs, cols=K,
                        group_size=16 if scheme == "nvfp4" else 32)


@pytest.mark.parametrize("scheme,K", SIZES)
def test_recipe_gives_a_weight_that_the_calls_take(scheme, K):
    from fni8 import ops

    N = 40
    packed, raw, _ = checkpoint(N, K, scheme, K)
    qt = qtensor(packed, raw, scheme, K)
    assert ops._fp4_shape(qt, "linear") == (N, K)
    assert torch.equal(qt.data[:, : K // 2], packed) and not qt.data[:, K // 2:].any()


def test_pad_codes():
    from fni8.quant.fp4 import pad_codes

    full = torch.randint(0, 256, (3, 16), dtype=torch.uint8)
    assert torch.equal(pad_codes(full, 32), full)
    assert torch.equal(pad_codes(full.view(torch.int8), 32), full)
    # codes behind K are dropped: the other half of an odd K's last byte, whole bytes
    odd = pad_codes(full, 25)
    assert torch.equal(odd[:, :12], full[:, :12]) and torch.equal(odd[:, 12], full[:, 12] & 15) and not odd[:, 13:].any()
    assert torch.equal(pad_codes(full[:, :13], 25), odd) and torch.equal(pad_codes(odd, 25), odd)
    assert pad_codes(full, 33 - 32).shape == (3, 16)
    assert torch.equal(pad_codes(torch.cat((full, full), 1)[:, ::2], 32), torch.cat((full, full), 1)[:, ::2])
    for bad, K in ((full, 34), (full, 0), (full[0], 32), (full.float(), 8), (full.to(torch.int16), 8)):
        with pytest.raises(ValueError):
            pad_codes(bad, K)


def test_unpadded_codes_are_refused_with_the_way_out():
    import fni8
    from fni8 import ops
    from fni8.quant import fp4

    packed, raw, _ = checkpoint(8, 48, "nvfp4", 1)
    qt = fni8.QTensor(packed, fp4.scale_tiles(raw), scheme="nvfp4", row_scale=torch.ones(8), cols=48)
    with pytest.raises(ValueError, match="pad_codes"):
        ops._fp4_shape(qt, "linear")


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a B200")
@pytest.mark.parametrize("M", [1, 40, 200])
@pytest.mark.parametrize("scheme,K", SIZES)
def test_product_of_an_imported_weight(scheme, K, M):
    """Rows of codes whose blocks all reach 6: the quantiser returns them as they are, every sum is a multiple of 1/8
    below 2^21, so the product is exact but for its rounding to bf16."""
    import fni8

    N = 72
    packed, raw, values = checkpoint(N, K, scheme, K + M)
    w = qtensor(packed, raw, scheme, K).to(DEV)
    g = torch.Generator().manual_seed(M)
    x = GRID[torch.randint(0, 16, (M, K), generator=g)]
    x[:, ::16] = 6.0
    assert torch.equal(fni8.dequantize_fp4(w, torch.float32).cpu().double(), values)
    want = (x @ values.t()).to(torch.bfloat16)
    got = fni8.linear(x.to(torch.bfloat16).to(DEV), w).cpu()
    assert torch.equal(got, want)
