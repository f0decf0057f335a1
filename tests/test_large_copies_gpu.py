"""Operands of more rows than a copy's grid has threads for: its workgroups go on to the
next rows."""

import pytest
import torch

import tilec
from test_fp8_gpu import check_product, operand


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_off_16_bytes(dtype):
    R, K = (1 << 30) + 1000, 33
    tail, w = operand(300, K, "e4m3", 1, 1), operand(1, K, "e4m3", 1, 2)
    codes = torch.zeros((R, K), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # 33 bytes a row: copied
    scales = torch.ones((R, 1), device="cuda")
    first = 1 << 29  # where half of the rows begin
    for at in (0, first, R - 300):
        codes[at:at + 300], scales[at:at + 300] = tail[0], tail[1]
    got = tilec.ext.linear_fp8((codes, scales), w, dtype=dtype)
    del codes, scales
    for at in (0, first, R - 300):
        check_product(got[at:at + 300], tail, w, 1, 1)
        got[at:at + 300] = 0
    assert not got.any()
    del got
    torch.cuda.empty_cache()
