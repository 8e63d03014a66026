"""Infinite weights in the layer of a few tokens: what the definition in 64 bits makes infinite
is infinite, with its sign, what it makes NaN is NaN, and nothing else is either."""
import pytest
import torch

from moe64 import merged64, routed64
from pdscope_amd import ops
from test_gpu_few import Layer

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")

# H of as many groups of 128 inputs as eight waves take in turn, and of fewer; activations
# in registers and in LDS
HS = [256, 384, 1024, 1536, 2176, 3200, 4096]


def with_infinity(T, H, rep, part, sign, seed):
    """A layer of one expert picked by every token beside others, one of whose weights (in
    `part`, of one of the last inputs) is infinite."""
    I, E, k = 256, 4, 2
    lay = Layer(T, H, I, E, k, rep, bias=True, seed=seed)
    lay.bias[:] = torch.tensor([0.0, 0.0, 30.0, 0.0], device=DEV)
    row, col = I - 3, H - 17
    at = {"gate": row * H, "up": I * H + row * H}[part] + col
    if rep == "bf16":
        lay.experts[2, at] = sign * INF
    else:
        n = 3 * I * H
        g = torch.Generator(device=DEV).manual_seed(seed)
        codes = torch.randint(0, 256, (E, n // 2), generator=g, device=DEV, dtype=torch.uint8)
        scales = torch.randint(118, 122, (E, n // 32), generator=g, device=DEV, dtype=torch.uint8)
        codes[2, at // 32 * 16:at // 32 * 16 + 16] = 0
        codes[2, at // 2] = (7 if sign > 0 else 15) << 4 * (at % 2)  # 6 times 2^127 is infinite in bf16
        scales[2, at // 32] = 254
        lay.blocks = ops.mxfp4_pack(codes, scales, H, I)
        lay.experts = ops.mxfp4_dequantize(lay.blocks, H, I)
        lay.slots = ops.slot_table([lay.blocks[e] for e in range(E)], DEV)
    assert torch.isinf(lay.experts).sum() == 1 and float(lay.experts[2, at]) == sign * INF
    return lay, row


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
@pytest.mark.parametrize("part", ["gate", "up"])
@pytest.mark.parametrize("H", HS)
def test_an_infinite_weight(H, part, rep):
    for T, sign in ((1, 1), (5, -1), (16, 1)):
        lay, row = with_infinity(T, H, rep, part, sign, seed=H + T)
        out, logits, ids, w = lay.run()
        x = lay.x.double()
        _, want_ids, _ = routed64(x, lay.gate.double(), lay.bias, lay.k, True)
        assert torch.equal(ids.long(), want_ids) and (ids == 2).any(1).all()
        want, _ = merged64(x, want_ids, w.double(), lay.block_of, lay.H, lay.I)
        # a picked expert's weight 0 (behind a bias of 30) times an infinite row is NaN in both
        assert torch.equal(torch.isnan(out), torch.isnan(want)), (T, sign)
        inf = torch.isinf(want)
        assert torch.equal(torch.isinf(out), inf) and torch.equal(out[inf].double(), want[inf])
        assert (inf | torch.isnan(want)).all()
