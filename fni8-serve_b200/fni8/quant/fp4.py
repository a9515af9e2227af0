"""Block scales of 4-bit floating point weights: rows to the kernels' tile order and back.

A checkpoint stores one scale byte per block in rows [N, S] (S = in_features / 32 e8m0 bytes
for MXFP4, / 16 e4m3 bytes for NVFP4). The block-scaled GEMM reads them in tiles of 128 rows
x 4 scales, 512 bytes each, in which row r and scale s are at byte (r % 32) * 16 +
(r % 128 / 32) * 4 + s % 4 (include/fni8_b200.h). A weight loaded from such a checkpoint is

    QTensor(pad_codes(packed, K), scale_tiles(rows), scheme="nvfp4", group_size=16, row_scale=..., cols=K)

with `packed` uint8 [N, K / 2], the even element in the low half; the kernels' rows have Kp / 2
bytes, Kp = K rounded up to 32, with zero codes behind K. Runs on any device; done once when a
model is loaded.
"""
from __future__ import annotations

import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pad_codes(codes: torch.Tensor, K: int) -> torch.Tensor:
    """Packed codes of K columns, uint8 [N, ceil(K / 2)] or wider, -> [N, Kp / 2] with Kp = K
    rounded up to 32, zero codes behind K. Codes that have this form already come back as they are."""
    if codes.dim() != 2 or codes.element_size() != 1 or codes.dtype.is_floating_point:
        raise ValueError("pad_codes: packed codes, one byte for two columns, [N, K / 2]")
    used, width = (K + 1) // 2, (K + 31) // 32 * 16
    if K < 1 or codes.shape[1] < used:
        raise ValueError(f"pad_codes: {tuple(codes.shape)} does not hold {K} columns")
    b = codes.contiguous().view(torch.uint8)
    if b.shape[1] == width and not (b[:, used:].any() or (K % 2 and (b[:, used - 1] >> 4).any())):
        return b
    out = torch.zeros(b.shape[0], width, dtype=torch.uint8, device=b.device)
    out[:, :used] = b[:, :used]
    if K % 2:
        out[:, used - 1] &= 15
    return out


def scale_tiles(rows: torch.Tensor) -> torch.Tensor:
    """Scale bytes [N, S] -> tiles uint8 [ceil(N / 128), ceil(S / 4), 512], zeros outside."""
    if rows.dim() != 2 or rows.element_size() != 1:
        raise ValueError("scale_tiles: one byte per block, [N, S]")
    b = rows.contiguous().view(torch.uint8)
    N, S = b.shape
    rt, st = (N + 127) // 128, (S + 3) // 4
    full = torch.zeros(rt * 128, st * 4, dtype=torch.uint8, device=b.device)
    full[:N, :S] = b
    return full.view(rt, 4, 32, st, 4).permute(0, 3, 2, 1, 4).reshape(rt, st, 512).contiguous()


def scale_rows(tiles: torch.Tensor, N: int, S: int) -> torch.Tensor:
    """Inverse of scale_tiles: the scale bytes [N, S] of the first N rows and S blocks."""
    if tiles.dim() != 3 or tiles.shape[2] != 512 or tiles.shape[0] * 128 < N or tiles.shape[1] * 4 < S:
        raise ValueError(f"scale_rows: {tuple(tiles.shape)} does not hold [{N}, {S}]")
    rt, st = tiles.shape[:2]
    return tiles.view(rt, st, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, st * 4)[:N, :S].contiguous()
