"""The routed experts of a prompt over 4-bit blocks (layer.experts_resident and moe_forward with
representation="mxfp4") against their definition in 64 bits, and a stack of blocks that
uses all of the 4-bit path together."""
import pytest
import torch

from moe64 import assert_within, merged64, routed64
from pdscope_amd import layer, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def make(T, H, I, E, k, *, seed=1, used=None):
    """Random 4-bit experts and a routing over the first `used` of them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    blocks = ops.mxfp4_quantize((0.05 * n(E, 3 * I * H)).to(BF16), H, I)
    x = n(T, H).to(BF16)
    scores = n(T, E) + n(E)
    if used is not None:
        scores[:, used:] = -1e9
    w, ids = torch.topk(torch.softmax(scores, 1), k, dim=1)
    return x, ids.to(torch.int32), w.to(BF16), blocks, ops.slot_table([blocks[e] for e in range(E)], DEV)


def check(out, x, ids, w, blocks, H, I, add_in=None, slots=None):
    values = ops.mxfp4_dequantize(blocks, H, I)
    want, bound = merged64(x.double(), ids.long(), w.double(),
                           lambda e: values[e].double() if slots is None or int(slots[e]) else None, H, I,
                           None if add_in is None else add_in.double(), rounded_rows=True)
    assert_within(out, want, bound)


# one row; experts of one row, of a tile's rows and one more; H and I of one input group, of odd
# numbers of them, H off a multiple of 256; the shapes of the framework's layers
@pytest.mark.parametrize("T,H,I,E,k", [(1, 128, 128, 1, 1), (2, 256, 128, 4, 2), (17, 128, 384, 8, 3), (33, 384, 128, 3, 1),
                                       (129, 640, 256, 2, 2), (65, 2048, 768, 128, 8), (700, 1024, 512, 64, 4),
                                       (301, 2048, 1408, 64, 6), (1025, 1536, 384, 96, 6), (600, 896, 640, 5, 2)])
def test_experts_of_a_prompt(T, H, I, E, k):
    x, ids, w, blocks, slots = make(T, H, I, E, k, seed=T)
    ws = layer.MoEWorkspace(T, H, I, E, k, DEV)
    out = layer.experts_resident(x, ids, w, slots, ws, representation="mxfp4")
    check(out, x, ids, w, blocks, H, I)


@pytest.mark.parametrize("block_m", [32, 64])
@pytest.mark.parametrize("T,used", [(5, 2), (130, 2), (257, 5), (515, 9)])
def test_every_row_tile_and_merge(block_m, T, used):
    """Experts of 1 to several hundred rows on each tile height: full tiles, every fill of
    the last one, experts without rows."""
    H, I, E, k = 512, 256, 12, 2
    x, ids, w, blocks, slots = make(T, H, I, E, k, seed=T + block_m, used=used)
    ws = layer.MoEWorkspace(T, H, I, E, k, DEV)
    add_in = torch.randn((T, H), device=DEV).to(BF16)
    out = layer.experts_resident(x, ids, w, slots, ws, block_m=block_m, add_in=add_in, representation="mxfp4")
    check(out, x, ids, w, blocks, H, I, add_in)
    again = layer.experts_resident(x, ids, w, slots, ws, out=torch.empty_like(out), block_m=block_m, add_in=add_in,
                                   representation="mxfp4")
    assert torch.equal(out, again)


def test_rows_counts_of_one_expert():
    """One expert with every count of rows around the tiles' edges."""
    H, I = 256, 128
    for block_m in (32, 64):
        for T in (1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 97, 113, 127, 128, 129):
            x, ids, w, blocks, slots = make(T, H, I, 1, 1, seed=T)
            ws = layer.MoEWorkspace(T, H, I, 1, 1, DEV)
            check(layer.experts_resident(x, ids, w, slots, ws, block_m=block_m, representation="mxfp4"), x, ids, w,
                  blocks, H, I)


def test_rows_of_an_expert_without_a_copy_are_kept():
    """As in the bf16 path: its rows of y are another launch's, and no other row is written."""
    T, H, I, E, k = 40, 256, 128, 4, 2
    x, ids, w, blocks, slots = make(T, H, I, E, k, seed=3)
    gone = int(torch.bincount(ids.flatten().long()).argmax())  # the expert of most rows
    slots[gone] = 0
    ws = layer.MoEWorkspace(2 * T, H, I, E, k, DEV)
    ws.y.fill_(7.0)
    layer.experts_resident(x, ids, w, slots, ws, representation="mxfp4")
    _, _, _, packed = ws.views(T)
    y = ws.y.view(-1, H)
    a, b = int(packed.offsets[gone]), int(packed.offsets[gone + 1])
    assert b > a and (y[a:b] == 7.0).all() and (y[T * k:] == 7.0).all()
    assert (y[:a] != 7.0).any(1).all() and (y[b:T * k] != 7.0).any(1).all()


@pytest.mark.parametrize("T,few", [(1, True), (16, True), (1, False), (9, False), (17, True), (200, False)])
@pytest.mark.parametrize("shared", [False, True])
def test_whole_layer(T, few, shared):
    H, I, E, k, Is = 512, 256, 32, 4, 384
    g = torch.Generator(device=DEV).manual_seed(T)
    x, _, _, blocks, slots = make(T, H, I, E, k, seed=T)
    gate = (0.05 * torch.randn((E, H), generator=g, device=DEV)).to(BF16)
    ws = layer.MoEWorkspace(T, H, I, E, k, DEV, shared_I=Is if shared else None, few_tokens=few)
    slot = sh = None
    if shared:
        sh = (0.05 * torch.randn(3 * Is * H, generator=g, device=DEV)).to(BF16)
        slot = ops.slot_table([sh], DEV)
    out, logits, ids, w = layer.moe_forward(x, gate, slots, ws, shared_slot=slot, representation="mxfp4")
    want_logits, want_ids, _ = routed64(x.double(), gate.double(), None, k, True)
    if few and T <= ops.FEW_MAX_TOKENS:
        assert torch.equal(logits, want_logits) and torch.equal(ids.long(), want_ids)
    add_in = None if sh is None else layer.shared_forward(x, slot, ws)
    check(out, x, ids, w, blocks, H, I, add_in)


def test_four_bit_stack_of_blocks():
    """Quantise two layers, run a prompt and then decode tokens through both, with the norms
    between blocks: every step against 64 bits on the inputs it was given."""
    H, I, E, k, L = 512, 384, 32, 3, 2
    g = torch.Generator(device=DEV).manual_seed(12)
    n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    experts = [(0.05 * n(E, 3 * I * H)).to(BF16) for _ in range(L)]
    blocks = [ops.mxfp4_quantize(e, H, I) for e in experts]
    values = [ops.mxfp4_dequantize(b, H, I).double() for b in blocks]
    slots = [ops.slot_table([b[e] for e in range(E)], DEV) for b in blocks]
    gates = [(0.05 * n(E, H)).to(BF16) for _ in range(L)]
    post, pre = [(1 + 0.1 * n(H)).to(BF16) for _ in range(L)], [(1 + 0.1 * n(H)).to(BF16) for _ in range(L)]
    ws = layer.MoEWorkspace(150, H, I, E, k, DEV, few_tokens=True)
    for T in (150, 1, 5, 16):
        resid, x = n(T, H), n(T, H).to(BF16)
        for l in range(L):
            out, _, ids, w = layer.moe_forward(x, gates[l], slots[l], ws, representation="mxfp4")
            want, bound = merged64(x.double(), ids.long(), w.double(), lambda e: values[l][e], H, I,
                                   rounded_rows=T > ops.FEW_MAX_TOKENS)
            assert_within(out, want, bound)
            r, x = ops.norm_residual(out, resid, post_weight=post[l], scale=0.7, pre_weight=pre[l])
            a = out.double()
            a = a / (a.square().mean(1, keepdim=True) + 1e-6).sqrt() * post[l].double()
            want = resid.double() + 0.7 * a
            # H + 8 roundings of the mean square, halved by the root, and four of the products
            assert_within(r, want, (H + 16) * 2.0 ** -24 * (want.abs() + a.abs()))
            m = r.double() / (r.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * pre[l].double()
            assert_within(x, m, (2.0 ** -8 + 2 * (H + 16) * 2.0 ** -24) * m.abs())
            if T > ops.FEW_MAX_TOKENS:  # the merge fused with the norms gives the same, unrounded in between
                _, _, _, packed = ws.views(T)
                r2, _ = ops.merge_norm_residual(ws.y, packed.row_of, w, resid, scale=0.7)
                want = resid.double() + 0.7 * out.double()
                assert_within(r2, want, 2.0 ** -8 * out.double().abs() + 16 * 2.0 ** -24 * (want.abs() + out.double().abs()))
            resid = r


def test_replay_of_a_prompt():
    T, H, I, E, k = 96, 512, 256, 16, 4
    x, ids, w, blocks, slots = make(T, H, I, E, k, seed=21)
    ws = layer.MoEWorkspace(T, H, I, E, k, DEV)
    want = layer.experts_resident(x, ids, w, slots, ws, representation="mxfp4").clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.experts_resident(x, ids, w, slots, ws, representation="mxfp4")
    for _ in range(3):
        got.zero_()
        ws.y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_rows_past_2_to_the_32_values():
    """2.2 million tokens, whose h has 4.5e9 values: tokens of the first rows, the last and some
    between have what a call over them alone gives (a row's products do not depend on
    the rows beside it)."""
    T, H, I, E, k = 2_200_000, 128, 1024, 4, 2
    x, ids, w, blocks, slots = make(T, H, I, E, k, seed=31)
    ws = layer.MoEWorkspace(T, H, I, E, k, DEV)
    assert ws.h_ws.numel() > 2 ** 32
    out = layer.experts_resident(x, ids, w, slots, ws, block_m=64, representation="mxfp4")
    pick = torch.cat([torch.arange(50), torch.arange(T // 2, T // 2 + 50), torch.arange(T - 50, T)]).to(DEV)
    few = layer.MoEWorkspace(pick.numel(), H, I, E, k, DEV)
    want = layer.experts_resident(x[pick], ids[pick], w[pick], slots, few, block_m=64, representation="mxfp4")
    assert torch.equal(out[pick], want)
    check(want, x[pick], ids[pick], w[pick], blocks, H, I)


def test_refusals():
    T, H, I, E, k = 20, 256, 128, 4, 2
    x, ids, w, blocks, slots = make(T, H, I, E, k)
    ws = layer.MoEWorkspace(T, H, I, E, k, DEV)
    with pytest.raises(ValueError, match="representation"):
        layer.experts_resident(x, ids, w, slots, ws, representation="fp8")
    with pytest.raises(ValueError, match="block_m"):
        layer.experts_resident(x, ids, w, slots, ws, block_m=128, representation="mxfp4")
    with pytest.raises(ValueError, match="add_in"):
        layer.experts_resident(x, ids, w, slots, ws, shared_slot=slots[:1], representation="mxfp4")
    with pytest.raises(ValueError, match="H % 128"):
        bad = layer.MoEWorkspace(T, 192, I, E, k, DEV)
        layer.experts_resident(x[:, :192].contiguous(), ids, w, slots, bad, representation="mxfp4")
    with pytest.raises(ValueError, match="next-layer prediction"):
        layer.moe_forward(x[:1], torch.zeros((E, H), dtype=BF16, device=DEV), slots, ws,
                          next_gate=torch.zeros((E, H), dtype=BF16, device=DEV),
                          pred_out=torch.zeros(k, dtype=torch.int32, device=DEV), representation="mxfp4")
    with pytest.raises(ValueError, match="inputs must be"):
        ops.swiglu_grouped_mxfp4(x[:, :128].contiguous(), ws.perm_token, ws.offsets, ws.sel_all, ws.tile_start, 4, 32,
                                 slots, H, I, ws.h_ws, ws.y)
