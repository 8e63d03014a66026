"""4-bit expert blocks: quantisation, decoding and checkpoint import.

The oracle is the format's definition in 64 bits on the CPU: a block of 32 inputs
has the scale 2^(floor(log2 of its largest magnitude) - 2), values go to the
nearest of the eight magnitudes, ties to the even code, above 6 to 6.  Everything
is compared for equality: no step of it rounds differently in fp32.
"""
import pytest
import torch

from pdscope_amd import ops

pytestmark = pytest.mark.gpu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize64(w):
    """Codes (0..15) and scale bytes of w [.., K] (finite bf16), on the CPU in fp64."""
    b = w.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = torch.where(top > 0, torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - 2, torch.tensor(-127.0, dtype=torch.float64))
    e = e.clamp(-127, 127)
    v = b.abs() * torch.exp2(-e).unsqueeze(-1)
    code = torch.zeros_like(v, dtype=torch.int64)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        code += (v > mid) | ((v == mid) & (i % 2 == 1))
    code += 8 * torch.signbit(b)
    return code.flatten(-2), (e + 127).to(torch.int64)


def values64(code, byte):
    v = GRID[code & 7] * torch.where(code >= 8, -1.0, 1.0).double()
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(byte.double() - 127).unsqueeze(-1)).flatten(-2)


def experts_like(kind, E, n, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((E, n), generator=g)
    if kind == "wide":  # magnitudes over the whole range of bf16, subnormal ones among them
        w = w * torch.exp2(torch.randint(-132, 126, (E, n // 32), generator=g).float()).repeat_interleave(32, 1)
    elif kind == "ties":  # multiples of an eighth: midpoints between neighbours are frequent
        w = torch.round(w * 16) / 8
    elif kind == "zeros":
        w = w * (torch.rand((E, n // 32), generator=g) < 0.5).float().repeat_interleave(32, 1)
        w[:, ::7] = -0.0
    return w.to(torch.bfloat16)


@pytest.mark.parametrize("kind", ["normal", "wide", "ties", "zeros"])
@pytest.mark.parametrize("E,H,I", [(1, 128, 128), (3, 256, 384), (2, 640, 128), (1, 2048, 768)])
def test_quantize_and_back(kind, E, H, I):
    w = experts_like(kind, E, 3 * I * H, 11 * E + H + I)
    blocks = ops.mxfp4_quantize(w.cuda(), H, I)
    assert tuple(blocks.shape) == (E, 3 * I * H * 17 // 32) and blocks.dtype == torch.uint8
    back = ops.mxfp4_dequantize(blocks, H, I).cpu().double()
    code, byte = quantize64(w)
    assert torch.equal(back, values64(code, byte))


@pytest.mark.parametrize("E,H,I", [(1, 128, 128), (5, 384, 256), (2, 1024, 512)])
def test_pack_of_a_checkpoint(E, H, I):
    """Random codes and scales, every byte value: the values come back, and the
    blocks equal those of quantising them where that is lossless."""
    n = 3 * I * H
    g = torch.Generator().manual_seed(E + H)
    codes = torch.randint(0, 256, (E, n // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(0, 255, (E, n // 32), generator=g, dtype=torch.uint8)
    blocks = ops.mxfp4_pack(codes.cuda(), scales.cuda(), H, I)
    got = ops.mxfp4_dequantize(blocks, H, I).cpu()
    code = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).long()
    want = values64(code, scales.long()).to(torch.bfloat16)  # 6 * 2^127 is infinite in bf16 too
    assert torch.equal(got, want)
    w = experts_like("normal", E, n, 5)
    code, byte = quantize64(w)
    blocks = ops.mxfp4_pack((code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8).cuda(), byte.to(torch.uint8).cuda(), H, I)
    assert torch.equal(blocks, ops.mxfp4_quantize(w.cuda(), H, I))


def test_infinities_and_nan_stay_in_their_block():
    """32 values with an infinity or NaN among them become NaN, and no others."""
    H, I = 128, 128
    w = experts_like("normal", 1, 3 * I * H, 3)
    for i, v in ((5, float("inf")), (70, float("nan")), (3 * I * H - 1, float("-inf"))):
        w[0, i] = v
    got = ops.mxfp4_dequantize(ops.mxfp4_quantize(w.cuda(), H, I), H, I).cpu()
    nan = torch.isnan(got)[0].view(-1, 32)
    want = torch.zeros(3 * I * H // 32, dtype=torch.bool)
    want[[0, 2, -1]] = True
    assert torch.equal(nan.all(1), want) and torch.equal(nan.any(1), want)


def test_more_than_2_to_the_32_weights():
    """1000 experts (4.7e9 weights), eight of them again and again: every block and every value
    equals the first eight's."""
    H, I, n, times = 2048, 768, 8, 125
    g = torch.Generator(device="cuda").manual_seed(7)
    some = (0.05 * torch.randn((n, 3 * I * H), generator=g, device="cuda")).to(torch.bfloat16)
    first = ops.mxfp4_quantize(some, H, I)
    blocks = ops.mxfp4_quantize(some.repeat(times, 1), H, I)
    assert blocks.shape[0] * 3 * I * H > 2 ** 32
    assert (blocks.view(times, n, -1) == first).all()
    values = ops.mxfp4_dequantize(blocks, H, I).view(torch.int16)
    want = ops.mxfp4_dequantize(first, H, I).view(torch.int16)
    for at in (0, 61 * n, (times - 1) * n):
        assert torch.equal(values[at:at + n], want)


def test_refusals():
    w = torch.zeros((2, 3 * 128 * 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="H % 128"):
        ops.mxfp4_quantize(w, 64, 128)
    with pytest.raises(ValueError, match="3\\*I\\*H"):
        ops.mxfp4_quantize(w, 128, 256)
    with pytest.raises(ValueError, match="must be torch.bfloat16"):
        ops.mxfp4_quantize(w.float(), 128, 128)
    with pytest.raises(ValueError, match="out must be"):
        ops.mxfp4_quantize(w, 128, 128, out=torch.empty((1, 4), dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="blocks must be"):
        ops.mxfp4_dequantize(torch.empty((2, 100), dtype=torch.uint8, device="cuda"), 128, 128)
    with pytest.raises(ValueError, match="scales"):
        ops.mxfp4_pack(torch.empty((2, 3 * 64 * 128), dtype=torch.uint8, device="cuda"),
                       torch.empty((2, 7), dtype=torch.uint8, device="cuda"), 128, 128)
    with pytest.raises(ValueError, match="contiguous"):
        ops.mxfp4_quantize(torch.zeros((2, 6 * 128 * 128), dtype=torch.bfloat16, device="cuda")[:, ::2], 128, 128)
    one = torch.zeros(3 * 128 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(1, -1)
    with pytest.raises(ValueError, match="alignment"):
        ops.mxfp4_quantize(one, 128, 128)
