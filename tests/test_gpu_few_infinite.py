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
    `part`, of one of the last inputs or columns) is infinite."""
    I, E, k = 256, 4, 2
    lay = Layer(T, H, I, E, k, rep, bias=True, seed=seed)
    lay.bias[:] = torch.tensor([0.0, 0.0, 30.0, 0.0], device=DEV)
    row, col = (I - 3, H - 17) if part != "down" else (H - 70, I - 3)
    at = {"gate": row * H, "up": I * H + row * H, "down": 2 * I * H + row * I}[part] + col
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
@pytest.mark.parametrize("part", ["gate", "up", "down"])
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
        if part == "down":  # one output of every token, the others as if the weight were 0
            assert inf[:, row].all() and int(inf.sum()) == T and not torch.isnan(want).any()
            finite = lay.experts.double()
            finite[torch.isinf(finite)] = 0
            want, bound = merged64(x, want_ids, w.double(), lambda e: finite[e], lay.H, lay.I)
            assert ((out.double() - want).abs() <= bound)[~inf].all()
        else:
            assert (inf | torch.isnan(want)).all()


def test_an_infinite_weight_against_h_of_one_bit():
    """h = silu(64) 0.5 = 32 everywhere: one bf16 part holds all of it."""
    H, I = 384, 256
    for T in (1, 16):
        lay, row = with_infinity(T, H, "bf16", "down", -1, seed=40)
        lay.x.zero_()
        lay.x[:, 0] = 1.0
        lay.experts[:, 0:I * H:H] = 64.0
        lay.experts[:, I * H:2 * I * H:H] = 0.5
        out, _, ids, w = lay.run()
        want, _ = merged64(lay.x.double(), ids.long(), w.double(), lay.block_of, H, I)
        assert (want[:, row] == -INF).all() and (out[:, row] == -INF).all()
        assert int(torch.isfinite(out).sum()) == T * (H - 1)
