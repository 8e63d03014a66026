"""The ends of what a 4-bit block can hold: values of 2^128 and more, which bf16 has not, are
infinite when they are decoded, the smallest ones are exact, and byte 255 makes NaN of all."""
import pytest
import torch

from pdscope_amd import ops
from test_gpu_mxfp4 import values64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("byte", [0, 1, 2, 252, 253, 254, 255])
def test_every_code_under_a_scale(byte):
    H = I = 128
    n = 3 * I * H
    code = torch.arange(n).remainder(16).view(1, n)
    codes = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
    scales = torch.full((1, n // 32), byte, dtype=torch.uint8)
    got = ops.mxfp4_dequantize(ops.mxfp4_pack(codes.cuda(), scales.cuda(), H, I), H, I).cpu().double()
    want = values64(code, scales.long())
    if byte == 255:
        assert torch.isnan(got).all()
        return
    large = want.abs() >= 2.0 ** 128
    assert int(large[0, :16].sum()) == {253: 4, 254: 8}.get(byte, 0)
    assert torch.equal(got[large], torch.copysign(torch.tensor(float("inf"), dtype=torch.float64), want[large]))
    assert torch.equal(got[~large], want[~large])
