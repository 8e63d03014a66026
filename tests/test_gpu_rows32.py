"""The experts' rows in fp32 between their down products and the merge: one rounding to bf16 in all.

With u = 2^-24, beside the bounds of test_gpu_grouped_mxfp8.py: a row y is its product's fp32 sum, off by ey;
the merge sums k of them in slot order, (k + 2) u of their magnitudes, and rounds: half a step of bf16."""
import pytest
import torch

from moe64 import assert_within
from pdscope_amd import layer, ops
from rows8 import rows8, values8
from test_gpu_grouped_mxfp8 import make, product

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
U, B = 2.0 ** -24, 2.0 ** -8


def check(out, ws, rows, ids, w, blocks, add_in=None, gone=()):
    """The rows against 64 bits on the hidden rows that were stored, and the output against the 64-bit
    sum of these 64-bit rows: a rounding in between would be off by up to 2^-8 of the summed magnitudes."""
    T, k = ids.shape
    H, I, E = ws.H, ws.I, ws.E
    values, packed = ops.mxfp4_dequantize(blocks, H, I), ws.views(T)[3]
    hv = values8(ops.MxRows(ws.h_rows().codes[:T * k], ws.h_rows().scales[:T * k]))
    y, off = ws.y.view(-1, H)[:T * k], packed.offsets.tolist()
    assert y.dtype is F32
    want, ey = torch.zeros((T * k, H), dtype=torch.float64, device=DEV), torch.zeros((T * k, H), dtype=torch.float64, device=DEV)
    for e in range(E):
        a, b = off[e], off[e + 1]
        if a < b and e not in gone:
            want[a:b], ey[a:b] = product(hv[a:b], values[e, 2 * I * H:].double().view(H, I))
            assert_within(y[a:b], want[a:b], ey[a:b])
    at, wd = packed.row_of.view(T, k).long(), w.double().unsqueeze(2)
    if gone:
        return
    total, mass, err = ((v[at] * wd).sum(1) for v in (want, want.abs(), ey))
    if add_in is not None:
        total, mass = total + add_in.double(), mass + add_in.double().abs()
    assert_within(out, total, (1 + B) * (err + (k + 2) * U * (mass + err)) + B * total.abs() + 2.0 ** -133)


def workspace(T, H, I, E, k, **kw):
    return layer.MoEWorkspace(T, H, I, E, k, DEV, y_dtype=F32, **kw)


@pytest.mark.parametrize("T,H,I,E,k", [(1, 128, 128, 1, 1), (2, 256, 128, 4, 2), (17, 128, 384, 8, 3), (33, 384, 128, 3, 1),
                                       (129, 640, 256, 2, 2), (65, 2048, 768, 128, 8), (700, 1024, 512, 64, 4),
                                       (301, 2048, 1408, 64, 6), (1025, 1536, 384, 96, 6), (40, 256, 128, 32, 12)])
@pytest.mark.parametrize("block_m", [None, 32, 64])
def test_experts(T, H, I, E, k, block_m):
    rows, ids, w, blocks, slots = make(T, H, I, E, k, seed=T)
    ws = workspace(T, H, I, E, k)
    add_in = torch.randn((T, H), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(BF16) if T % 2 else None
    out = layer.experts_resident(rows, ids, w, slots, ws, block_m=block_m, add_in=add_in, representation="mxfp4")
    check(out, ws, rows, ids, w, blocks, add_in)
    again = layer.experts_resident(rows, ids, w, slots, ws, out=torch.empty_like(out), block_m=block_m, add_in=add_in,
                                   representation="mxfp4")
    assert torch.equal(out, again)


def test_row_counts_of_one_expert():
    H, I = 256, 128
    for block_m in (32, 64):
        for T in (1, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 97, 113, 127, 128, 129):
            rows, ids, w, blocks, slots = make(T, H, I, 1, 1, seed=T)
            ws = workspace(2 * T, H, I, 1, 1)
            ws.y.fill_(7.0)
            out = layer.experts_resident(rows, ids, w, slots, ws, block_m=block_m, representation="mxfp4")
            check(out, ws, rows, ids, w, blocks)
            assert (ws.y.view(-1, H)[T:] == 7.0).all()


def test_rows_of_an_expert_without_a_copy_are_kept():
    T, H, I, E, k = 40, 256, 128, 4, 2
    rows, ids, w, blocks, slots = make(T, H, I, E, k, seed=3)
    gone = int(torch.bincount(ids.flatten().long()).argmax())
    slots[gone] = 0
    ws = workspace(2 * T, H, I, E, k)
    ws.y.fill_(7.0)
    out = layer.experts_resident(rows, ids, w, slots, ws, representation="mxfp4")
    off, y = ws.views(T)[3].offsets.tolist(), ws.y.view(-1, H)
    a, b = off[gone], off[gone + 1]
    assert b > a and (y[a:b] == 7.0).all() and (y[T * k:] == 7.0).all()
    check(out, ws, rows, ids, w, blocks, gone=(gone,))


def test_nan_rows_stay_their_own():
    T, H, I, E, k = 50, 256, 128, 3, 1
    rows, ids, w, blocks, slots = make(T, H, I, E, k, seed=4)
    ws = workspace(T, H, I, E, k)
    want = layer.experts_resident(rows, ids, w, slots, ws, representation="mxfp4").clone()
    bad = ops.MxRows(rows.codes, rows.scales.clone())
    bad.scales[7, 3] = 255
    out = layer.experts_resident(bad, ids, w, slots, ws, representation="mxfp4")
    keep = torch.arange(T, device=DEV) != 7
    assert torch.isnan(out[7]).all() and torch.equal(out[keep], want[keep])


@pytest.mark.parametrize("T", [1, 9, 200])
def test_layer_and_the_norm_behind_it(T):
    """moe_forward on such a workspace, and the merge of its rows with the next norm."""
    H, I, E, k = 512, 256, 32, 4
    g = torch.Generator(device=DEV).manual_seed(T)
    n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    _, _, _, blocks, slots = make(T, H, I, E, k, seed=T)
    x, gate, pre = n(T, H).to(BF16), (0.05 * n(E, H)).to(BF16), (1 + 0.1 * n(H)).to(BF16)
    ws = workspace(T, H, I, E, k, mxfp8=True)
    out, _, ids, w = layer.moe_forward(x, gate, slots, ws, representation="mxfp4", activations="mxfp8")
    check(out, ws, ops.mxfp8_quantize(x), ids, w, blocks)
    before = n(T, H)
    resid, norm, rows = ops.merge_norm_residual(ws.y, ws.views(T)[3].row_of, w, before, pre_weight=pre, want_mxfp8=True)
    at = ws.views(T)[3].row_of.view(T, k).long()
    r = before.double() + (ws.y.view(-1, H).double()[at] * w.double().unsqueeze(2)).sum(1)
    assert_within(resid, r, U * (1 + 2.0 ** -20) * r.abs() + 2.0 ** -40)
    m = r / (r.square().mean(1, keepdim=True) + float(torch.tensor(1e-6, dtype=F32))).sqrt() * pre.double()
    assert_within(norm, m, B * (1 + 2.0 ** -20) * m.abs())
    assert torch.equal(values8(rows), rows8(m)[2])


def rows32(T, H, k, seed, extra=3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    y = torch.randn((T * k + extra, H), generator=g, device=DEV)
    at = torch.randperm(T * k + extra, generator=g, device=DEV)[:T * k].to(torch.int32)
    w = torch.softmax(torch.randn((T, k), generator=g, device=DEV), 1).to(BF16)
    return y, at, w, torch.randn((T, H), generator=g, device=DEV).to(BF16)


@pytest.mark.parametrize("T,H,k", [(1, 8, 1), (3, 24, 2), (5, 1504, 7), (2, 2048, 8), (130, 2048, 8), (9, 520, 9), (33, 1024, 16),
                                   (4, 96, 17), (70, 264, 20), (1000, 512, 6)])
@pytest.mark.parametrize("summand", [False, True])
def test_merge(T, H, k, summand):
    y, at, w, add_in = rows32(T, H, k, seed=T + k)
    out = ops.merge(y.flatten(), at, w, torch.empty((T, H), dtype=BF16, device=DEV), add_in=add_in if summand else None)
    terms = y.double()[at.view(T, k).long()] * w.double().unsqueeze(2)
    want, mass = terms.sum(1), terms.abs().sum(1)
    if summand:
        want, mass = want + add_in.double(), mass + add_in.double().abs()
    assert_within(out, want, (1 + B) * (k + 2) * U * mass + B * want.abs())


@pytest.mark.parametrize("T,H,k", [(1, 2048, 8), (3, 64, 1), (17, 1504, 6), (130, 2048, 8), (2, 16384, 3), (4, 37, 5), (2, 9001, 2)])
@pytest.mark.parametrize("R,P", [(BF16, BF16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("offset", [0, 1])
def test_merge_and_norm(T, H, k, R, P, offset):
    """Rows of fp32, aligned and not, rows that are not there; with 8-bit rows and without."""
    y, at, w, add_in = rows32(T, H, k, seed=T + H)
    room = torch.empty(y.numel() + offset, device=DEV)
    room[offset:] = y.flatten()
    at[0], at[-1] = -1, y.shape[0]
    g = torch.Generator(device=DEV).manual_seed(k)
    resid = (2 * torch.randn((T, H), generator=g, device=DEV)).to(R)
    pre = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(P)
    args = dict(add_in=add_in, pre_weight=pre, scale=0.75)
    r, n = ops.merge_norm_residual(room[offset:], at, w, resid, **args)
    idx = at.view(T, k).long()
    ok = ((idx >= 0) & (idx < y.shape[0])).double()
    terms = y.double()[idx.clamp(0, y.shape[0] - 1)] * (w.double() * ok).unsqueeze(2)
    a, mass = terms.sum(1) + add_in.double(), terms.abs().sum(1) + add_in.double().abs()
    wr = resid.double() + 0.75 * a
    rms = (wr.square().mean(1, keepdim=True) + float(torch.tensor(1e-6, dtype=F32))).sqrt()
    wn = wr / rms * pre.double()
    half = U if R is F32 else B
    er = (k + 4) * U * (mass + resid.double().abs())
    assert_within(r, wr, (1 + half) * er + half * wr.abs())
    # the mean square is off by (H + 2) u and twice er, the root by half of that, the products by 3 roundings
    assert_within(n, wn, (1 + B) * (1.1 * er / rms * pre.double().abs() + (H + 8) * U * wn.abs()
                                    + 1.1 * (er * wr.abs()).mean(1, keepdim=True) / rms ** 2 * wn.abs()) + B * wn.abs())
    if H % 32 == 0:
        r, n, rows = ops.merge_norm_residual(room[offset:], at, w, resid, want_mxfp8=True, **args)
        assert_within(r, wr, half * (1 + 2.0 ** -30) * wr.abs() + 2.0 ** -38)
        assert_within(n, wn, B * (1 + 2.0 ** -30) * wn.abs() + 2.0 ** -38)
        assert torch.equal(values8(rows), rows8(wn)[2])


def test_replay_and_another_stream():
    T, H, I, E, k = 96, 512, 256, 16, 4
    rows, ids, w, blocks, slots = make(T, H, I, E, k, seed=21)
    ws = workspace(T, H, I, E, k)
    want = layer.experts_resident(rows, ids, w, slots, ws, representation="mxfp4").clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer.experts_resident(rows, ids, w, slots, ws, out=torch.empty_like(want), representation="mxfp4")
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.experts_resident(rows, ids, w, slots, ws, representation="mxfp4")
    for _ in range(3):
        for t in (got, ws.y, ws.h_ws):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_rows_past_2_to_the_32_bytes():
    """1.1 million tokens, whose rows have 9.0e9 bytes: tokens of the first rows, the last and some
    between have what a call over them alone gives."""
    T, H, I, E, k = 1_100_000, 1024, 128, 4, 2
    rows, ids, w, blocks, slots = make(T, H, I, E, k, seed=31)
    ws = workspace(T, H, I, E, k)
    out = layer.experts_resident(rows, ids, w, slots, ws, block_m=64, representation="mxfp4")
    pick = torch.cat([torch.arange(50), torch.arange(T // 2, T // 2 + 50), torch.arange(T - 50, T)]).to(DEV)
    few = workspace(pick.numel(), H, I, E, k)
    some = ops.MxRows(rows.codes.view(torch.uint8)[pick].view(ops.F8), rows.scales[pick])
    want = layer.experts_resident(some, ids[pick], w[pick], slots, few, block_m=64, representation="mxfp4")
    assert torch.equal(out[pick], want)
    check(want, few, some, ids[pick], w[pick], blocks)


def test_refusals():
    T, H, I, E, k = 20, 256, 128, 4, 2
    rows, ids, w, blocks, slots = make(T, H, I, E, k)
    ws = workspace(T, H, I, E, k)
    x = ops.mxfp8_dequantize(rows)
    with pytest.raises(ValueError, match="y_dtype"):
        layer.MoEWorkspace(T, H, I, E, k, DEV, y_dtype=torch.float16)
    with pytest.raises(ValueError, match="fp32 rows"):  # rows of bf16 products are bf16
        layer.experts_resident(x, ids, w, slots, ws, representation="mxfp4")
    with pytest.raises(ValueError, match="fp32 rows"):
        layer.experts_resident(x, ids, w, slots, ws)
    with pytest.raises(ValueError, match="fp32 rows"):
        layer.experts_resident(rows, ids, w, slots, ws, representation="mxfp4", merge="reference")
    with pytest.raises(ValueError, match="mode 'fused'"):
        ops.merge(ws.y, ws.row_of, w, ws.out, mode="reference")
    with pytest.raises(ValueError, match="y must be"):
        ops.merge(ws.y.double(), ws.row_of, w, ws.out)
    with pytest.raises(ValueError, match="y must be"):
        ops.merge_norm_residual(ws.y.half(), ws.row_of, w, x)
    with pytest.raises(ValueError, match="smaller than"):
        ops.swiglu_grouped_mxfp8(rows, ws.perm_token, ws.offsets, ws.sel_all, ws.tile_start, 4, 32, slots, H, I, ws.h_rows(),
                                 ws.y[:-1].contiguous())
    gate = torch.zeros((E, H), dtype=BF16, device=DEV)
    with pytest.raises(ValueError):
        layer.moe_forward(x, gate, slots, ws, representation="mxfp4")
