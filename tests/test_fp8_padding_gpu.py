"""The bytes between a row's last code and the next multiple of 16: zeros, whatever the
row holds, from both writers of 8-bit rows."""

import pytest
import torch

import tilec

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
WIDE = {"f32": torch.float32, "bf16": torch.bfloat16}
SHAPES = [(1, 7), (5, 129), (130, 257), (300, 400), (129, 16), (40, 511), (260, 1)]


def rows_of(codes):
    """The bytes that the rows of codes [R, C] take in memory, [R, C up to 16]."""
    R, C = codes.shape
    room = -(-C // 16) * 16
    assert R == 1 or codes.stride(0) == room
    return codes.view(torch.uint8).as_strided((R, room), (room, 1)).cpu()


def values(R, C, dtype, bad):
    x = torch.randn(R, C, generator=torch.Generator().manual_seed(R + C))
    if bad is not None:  # in the last block of a row, and of a tile
        x[R // 2, C - 1] = bad
        x[R - 1, C - 1] = bad
    return x.to(WIDE[dtype]).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,to", [("f32", "e4m3"), ("bf16", "e4m3"), ("f32", "e5m2"), ("bf16", "e5m2")])
@pytest.mark.parametrize("bad", [None, float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("R,C", SHAPES)
def test_quantised_rows_end_in_zeros(R, C, bad, dtype, to):
    x = values(R, C, dtype, bad)
    sources = {"rows": x, "transposed": x.t().contiguous().t() if R > 1 and C > 1 else x}
    for name, s in sources.items():
        for block in (1, 128):
            codes, scales = tilec.ext.quantize_fp8(s, (block, 128), F8[to])
            got = rows_of(codes)
            assert (got[:, C:] == 0).all(), (name, block)
            # The codes themselves: NaNs where the block has no scale, the values' elsewhere.
            each = scales.repeat_interleave(block, 0)[:R].repeat_interleave(128, 1)[:, :C]
            assert torch.equal(torch.isnan(codes.float()), torch.isnan(each)), (name, block)
            assert bool(torch.isnan(each).any()) == (bad is not None), (name, block)


@pytest.mark.gpu
@pytest.mark.parametrize("to", list(F8))
@pytest.mark.parametrize("bad", [None, float("nan"), float("inf")])
@pytest.mark.parametrize("R,C", SHAPES)
def test_normalised_rows_end_in_zeros(R, C, bad, to):
    codes, scales = tilec.ext.rms_norm(values(R, C, "bf16", bad), dtype=F8[to])[0]
    assert (rows_of(codes)[:, C:] == 0).all()
    assert bool(torch.isnan(scales).any()) == (bad is not None)
