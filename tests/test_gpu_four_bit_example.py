"""The documented run over 4-bit experts, from quantising to the next block's input: the merge
inside the norms' launch gives what experts_resident and norm_residual give one after the
other, but for the rounding of the output between them."""
import pytest
import torch

from pdscope_amd import layer, ops

pytestmark = pytest.mark.gpu
U, B = 2.0 ** -24, 2.0 ** -8


@pytest.mark.parametrize("T", [1, 16, 17, 300])
def test_the_documented_run(T):
    H, I, E, k = 512, 256, 32, 4
    g = torch.Generator(device="cuda").manual_seed(T)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    bf = lambda t: t.to(torch.bfloat16)  # noqa: E731
    x, gate, experts, resid = bf(n(T, H)), bf(0.05 * n(E, H)), bf(0.05 * n(E, 3 * I * H)), n(T, H)
    w1, w2 = bf(1 + 0.1 * n(H)), bf(1 + 0.1 * n(H))
    blocks = ops.mxfp4_quantize(experts, H, I)
    slots = ops.slot_table([blocks[e] for e in range(E)], "cuda")
    ws = layer.MoEWorkspace(512, H, I, E, k, "cuda", few_tokens=True)
    out, logits, ids, weights = layer.moe_forward(x, gate, slots, ws, representation="mxfp4")
    if T <= ops.FEW_MAX_TOKENS:
        want = out.clone()
        out, _, ids, weights = layer.moe_few(x, gate, slots, ws, representation="mxfp4")
        assert torch.equal(out, want)
    out = layer.experts_resident(x, ids, weights, slots, ws, representation="mxfp4").clone()
    r1, n1 = ops.norm_residual(out, resid, post_weight=w1, scale=0.5, pre_weight=w2)

    ws.y.fill_(float("nan"))
    packed, bm = ws.views(T)[3], ops.grouped_mxfp4_block_m(T * k // E)
    ops.pack(ids, E, out=packed, workspace=ws.pack_ws, schedule=(ws.sel_all, bm, ws.sel_order, ws.tile_start))
    ops.swiglu_grouped_mxfp4(x, packed.perm_token, packed.offsets, ws.sel_order, ws.tile_start,
                             (T * k + bm - 1) // bm + E, bm, slots, H, I, ws.h_ws, ws.y)
    r2, n2 = ops.merge_norm_residual(ws.y, packed.row_of, weights, resid, post_weight=w1, scale=0.5, pre_weight=w2)

    # out is rounded before the first norm only: a value is off by B of itself, and the
    # root mean square, which divides all of them, by B at most
    a = out.double()
    a = 0.5 * a / (a.square().mean(1, keepdim=True) + 1e-6).sqrt() * w1.double()
    off = 2 * B * (1 + B) * a.abs() + (H + 16) * 2 * U * (a.abs() + resid.double().abs())
    assert ((r1.double() - r2.double()).abs() <= off).all()
    m = (r1.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    rel = (off.square().mean(1, keepdim=True).sqrt() / m) * (1 + B)
    want = r1.double() / m * w2.double()
    bound = (off / m) * w2.double().abs() * (1 + rel) + (2 * rel + 2 * B + (H + 16) * 2 * U) * want.abs()
    assert ((n1.double() - n2.double()).abs() <= bound).all()
