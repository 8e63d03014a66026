"""8-bit rows that calls make for themselves: the experts' hidden rows, taken together, and x quantised
in a layer's call.

A product of codes is off by about 4e-6 of its size (the matrix instruction's cuts).  A hidden value is a
product of two such, silu(g) u, and gets its neighbour's code where a border lies within its error e: of
all values a share of e / step, with steps of at least 1/16 of the value.  For normal g and u the mean of
1/|g| from 10^-3 of its spread on is 0.8 ln(10^3), 5.5 of it, and u's likewise: 16 (5.5 + 5.5) 4e-6 =
7e-4 of the values.  2^-7, eleven times that, is the limit here.  A value's neighbour is at most 1/8 of it
away, so that in a share of 2^-7 the difference has a norm of at most sqrt(2^-7) / 8 of the rows', and a
part along them of 2^-7 / 8 even if every one went the same way.  A loss of a thousandth in either
product would move some 12 thousandths of the values, cutting instead of rounding half of them."""
import pytest
import torch

from pdscope_amd import layer, ops
from rows8 import rows8, values8
from test_gpu_grouped_mxfp8 import make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.mark.parametrize("T,H,I,E,k", [(65, 2048, 768, 128, 8), (301, 2048, 1408, 64, 6), (700, 1024, 512, 64, 4),
                                       (400, 128, 384, 8, 3), (129, 640, 256, 2, 2)])
@pytest.mark.parametrize("block_m", [32, 64])
def test_hidden_rows_together(T, H, I, E, k, block_m):
    rows, ids, w, blocks, slots = make(T, H, I, E, k, seed=T + 7)
    ws = layer.MoEWorkspace(T, H, I, E, k, DEV)
    layer.experts_resident(rows, ids, w, slots, ws, block_m=block_m, representation="mxfp4")
    packed = ws.views(T)[3]
    h = ops.MxRows(ws.h_rows().codes[:T * k], ws.h_rows().scales[:T * k])
    x, values = values8(rows)[packed.perm_token.long()], ops.mxfp4_dequantize(blocks, H, I)
    want, off = torch.empty((T * k, I), dtype=torch.float64, device=DEV), packed.offsets.tolist()
    for e in range(E):
        a, b = off[e], off[e + 1]
        gate, up = (values[e, j * I * H:(j + 1) * I * H].double().view(I, H) for j in (0, 1))
        g = x[a:b] @ gate.T
        want[a:b] = g * torch.sigmoid(g) * (x[a:b] @ up.T)
    _, scales, rounded = rows8(want)
    got = values8(h)
    assert (h.scales != scales).double().mean() <= 2.0 ** -10
    assert (got != rounded).double().mean() <= 2.0 ** -7
    assert (got - rounded).norm() <= 2.0 ** -3.5 / 8 * rounded.norm()
    assert ((got - rounded) * rounded).sum().abs() <= 2.0 ** -10 * rounded.square().sum()


def test_rows_quantised_in_the_call():
    """x_rows left out: the layer runs on mxfp8_quantize(x), of this call's x and no other's."""
    H, I, E, k = 512, 256, 32, 4
    _, _, _, blocks, slots = make(1, H, I, E, k, seed=2)
    g = torch.Generator(device=DEV).manual_seed(11)
    gate = (0.05 * torch.randn((E, H), generator=g, device=DEV)).to(BF16)
    ws = layer.MoEWorkspace(300, H, I, E, k, DEV, mxfp8=True)
    other = layer.MoEWorkspace(300, H, I, E, k, DEV)
    for T in (300, 1, 9, 40, 299, 9):
        x = torch.randn((T, H), generator=g, device=DEV).to(BF16)
        out, logits, ids, w = layer.moe_forward(x, gate, slots, ws, representation="mxfp4", activations="mxfp8")
        rows = ops.mxfp8_quantize(x)
        assert torch.equal(ws.x_rows.codes[:T].view(torch.uint8), rows.codes.view(torch.uint8))
        assert torch.equal(ws.x_rows.scales[:T], rows.scales)
        want = layer.moe_forward(x, gate, slots, other, representation="mxfp4", activations="mxfp8", x_rows=rows)
        for a, b in zip((out, logits, ids, w), want):
            assert torch.equal(a, b)
