"""4-bit matrices at the ends of bf16's range: weights whose span is past fp32's largest number, and the
largest inputs of a product."""
import pytest
import torch

from pdscope_amd import ops
from test_gpu_int4 import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("top", [1.0, 1.6e38, 2.0e38, 2.9e38, 3.0 * 2.0 ** -130])
def test_spans_of_every_size(G, top):
    """s = bf16((max - min) / 15) with the span in 64 bits, which holds each quotient to 2^-52: the
    weights' eight bits lie on no border between two scales that a second rounding would cross (the
    test says so of its inputs), z and q are whole numbers next to the quotients by that scale."""
    N, K = 33, 512
    g = torch.Generator(device=DEV).manual_seed(G)
    weight = ((2 * torch.rand((N, K), generator=g, device=DEV, dtype=torch.float64) - 1) * top).to(BF16)
    w = ops.int4_quantize(weight, G, True)
    v = weight.double().unflatten(1, (-1, G))
    lo, hi = (-v).amax(2).clamp(min=0), v.amax(2).clamp(min=0)
    exact = (hi + lo) / 15
    s = exact.float().to(BF16)
    for side in (1 - 2.0 ** -22, 1 + 2.0 ** -22) if top > 1e-30 else ():
        assert torch.equal((exact * side).float().to(BF16), s)
    assert torch.isfinite(s.float()).all() and (s > 0).all()
    sd = s.double()
    z = torch.round(lo / sd)
    q = (torch.round(v / sd.unsqueeze(2)) + z.unsqueeze(2)).clamp(0, 15).flatten(1).to(torch.uint8)
    want = ops.int4_pack(q[:, 0::2] | (q[:, 1::2] << 4), s, z.to(torch.uint8))
    back, wanted = ops.int4_dequantize(w), ops.int4_dequantize(want)
    assert torch.isfinite(back.float()).all()
    assert torch.equal(back, wanted) and torch.equal(w.units, want.units)


@pytest.mark.parametrize("G", [32, 128])
@pytest.mark.parametrize("T,N", [(3, 100), (16, 105_001), (40, 1003), (200, 3001), (500, 4001), (1100, 4001), (2000, 4095)])
def test_inputs_up_to_2_to_the_117(T, N, G):
    """Whole groups of one sign at the largest magnitude below it, codes of 15 among them: a group's sum
    of q x is at most 15 G 2^117, below 2^128."""
    K = 1920
    g = torch.Generator(device=DEV).manual_seed(N)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    codes[::5] = 255
    scales = (0.002 + 0.01 * torch.rand((N, K // G), generator=g, device=DEV)).to(BF16)
    z = torch.randint(0, 16, (N, K // G), generator=g, device=DEV, dtype=torch.uint8)
    z[1::5] = 15
    x = torch.randn((T, K), generator=g, device=DEV).sign().mul(255 * 2.0 ** 109).to(BF16)
    x[0], x[T - 1] = 255 * 2.0 ** 109, -255 * 2.0 ** 109
    y = ops.linear_int4(x, ops.int4_pack(codes, scales, z))
    assert torch.isfinite(y.float()).all()
    check(y, x, codes, scales, z, G)
