"""Norms with 8-bit rows below fp32's normal numbers: one rounding there too.

fp32 has steps of 2^-149 below 2^-126, bf16 of 2^-133 and the codes of the smallest scale 2^-127 of at
least 2^-136: a value that went through the nearest fp32 number on its way is rounded twice, and once in
2^16 (bf16) or 2^14 (codes) times to another side of a border."""
import pytest
import torch

from pdscope_amd import ops
from rows8 import rows8, values8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def to_bf16(v):
    """fp64 values below 2^-126 as bf16, rounded once: whole steps of 2^-133, ties to even."""
    assert (v.abs() < 2.0 ** -126).all()
    return (torch.round(v * 2.0 ** 133) * 2.0 ** -133).to(BF16)


@pytest.mark.parametrize("positive", [True, False])
def test_a_sum_beside_a_border(positive):
    """resid + scale block is 49 steps of 2^-156 below the middle of two bf16 numbers, less than half a
    step of fp32: first above 0, then below it."""
    H = 64
    a, m = torch.tensor(137 / 128), 30615  # 137 m = 2^22 - 49
    block = torch.full((1, H), float(a), dtype=BF16, device=DEV)
    # (1 or -3) 2^-133 + (2^22 - 49) 2^-156: between 1 and 2 steps of 2^-133, nearer 1, or -3 and -2, nearer -3
    resid = want = 2.0 ** -133 if positive else -3 * 2.0 ** -133
    r = torch.full((1, H), resid, dtype=BF16, device=DEV)
    exact = resid + (2 ** 22 - 49) * 2.0 ** -156
    assert round(exact * 2.0 ** 133) * 2.0 ** -133 == want
    got, _, _ = ops.norm_residual(block, r, scale=m * 2.0 ** -149, want_mxfp8=True)
    assert (got.double() == want).all()


def test_norms_below_the_normal_numbers():
    T, H = 1024, 2048
    g = torch.Generator(device=DEV).manual_seed(3)
    n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    block, resid = n(T, H).to(BF16), (2 * n(T, H)).to(BF16)
    pre = (1 + 0.2 * n(H)) * 2.0 ** -130
    _, norm, rows = ops.norm_residual(block, resid, pre_weight=pre, want_mxfp8=True)
    r = resid.double() + block.double()
    want = r / torch.sqrt(r.square().mean(1, keepdim=True) + float(torch.tensor(1e-6, dtype=F32))) * pre.double()
    codes, scales, values = rows8(want)
    assert torch.equal(norm, to_bf16(want))
    assert torch.equal(rows.scales, scales) and torch.equal(values8(rows), values)
