"""4-bit matrices at the ends of bf16's range: weights whose span is past fp32's largest number."""
import pytest
import torch

from pdscope_amd import ops

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
