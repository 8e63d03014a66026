"""8-bit rows: conversions, and the norms between blocks that write them, against their definition
in 64 bits.  Codes and scales are compared bit for bit: the conversions' arithmetic is exact, and
the norms hold 64 bits, whose own error (some 1e-15) lies on a border between two codes for none
of the seeds here."""
import pytest
import torch

from moe64 import assert_within
from pdscope_amd import ops
from rows8 import rows8, values8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
B = 2.0 ** -8   # half a step of bf16
U = 2.0 ** -24  # and of fp32


def normal(*s, seed=1):
    return torch.randn(s, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def same(rows, v):
    codes, scales, values = rows8(v)
    assert torch.equal(rows.scales, scales)
    got = rows.codes.view(torch.uint8)
    assert torch.equal(got & 127, codes & 127)
    assert torch.equal(got, codes)
    assert torch.equal(values8(rows), values)


@pytest.mark.parametrize("T,n", [(1, 32), (1, 2048), (3, 96), (7, 1504), (33, 4096), (1000, 64), (5, 16416)])
@pytest.mark.parametrize("spread", [0.0, 8.0])
def test_quantise_and_back(T, n, spread):
    x = (normal(T, n, seed=T + n) * torch.exp2(spread * normal(T, n, seed=2))).to(BF16)
    rows = ops.mxfp8_quantize(x)
    same(rows, x.double())
    assert torch.equal(ops.mxfp8_dequantize(rows).double(), values8(rows))


def test_every_code_border_and_scale():
    """Each code, the midpoints between neighbours and their bf16 neighbours, at small, ordinary and
    large scales; blocks whose largest magnitude is 448 scales, a step below and above; zeros."""
    from rows8 import grid
    g = grid("cpu")
    v = torch.cat([g, (g[1:] + g[:-1]) / 2]).to(BF16)
    bits = v.view(torch.int16)
    v = torch.cat([v, (bits + 1).view(BF16), (bits[1:] - 1).view(BF16)])
    v = torch.cat([v, -v])
    v = v[v.abs() <= 448]
    blocks = []
    for top in (448.0, 450.0, 446.0, 256.0, 224.0):
        for part in torch.split(v[v.abs() <= top], 31):
            blocks.append(torch.cat([torch.tensor([top], dtype=BF16), part, torch.zeros(31 - len(part), dtype=BF16)]))
    x = torch.stack(blocks).to(DEV)
    x = torch.cat([x * 2.0 ** e for e in (-125, -118, -60, 0, 60, 118)])
    x = torch.cat([x, torch.zeros((1, 32), dtype=BF16, device=DEV)])
    x = x[torch.isfinite(x.float()).all(1)].contiguous()
    rows = ops.mxfp8_quantize(x)
    codes, scales, values = rows8(x.double())
    assert torch.equal(rows.scales, scales)
    assert torch.equal(values8(rows), values)
    big = values.abs() >= 2.0 ** -126
    assert torch.equal(torch.where(big, ops.mxfp8_dequantize(rows).double(), values), values)


def test_infinities_and_nan_make_their_block_nan():
    x = normal(4, 96).to(BF16)
    x[0, 5], x[1, 40], x[2, 95] = float("inf"), float("nan"), -float("inf")
    rows = ops.mxfp8_quantize(x)
    back = ops.mxfp8_dequantize(rows)
    want = torch.zeros((4, 3), dtype=torch.bool, device=DEV)
    want[0, 0] = want[1, 1] = want[2, 2] = True
    assert torch.equal(rows.scales == 255, want)
    assert torch.equal(torch.isnan(back).view(4, 3, 32), want.unsqueeze(2).expand(4, 3, 32))
    ok = ~want.repeat_interleave(32, 1)
    assert torch.equal(values8(rows)[ok], rows8(x.nan_to_num(0, 0, 0).double())[2][ok])


def test_no_rows():
    x = torch.empty((0, 64), dtype=BF16, device=DEV)
    rows = ops.mxfp8_quantize(x)
    assert rows.codes.shape == (0, 64) and ops.mxfp8_dequantize(rows).shape == (0, 64)


def test_past_2_to_the_31_values():
    T, n = 70_000, 32768
    x = torch.empty((T, n), dtype=BF16, device=DEV)
    x.copy_(normal(1, n, seed=4).to(BF16).expand(T, n))
    x[T - 1] = normal(1, n, seed=5).to(BF16)
    rows = ops.mxfp8_quantize(x)
    last = ops.MxRows(rows.codes[T - 1:], rows.scales[T - 1:])
    same(last, x[T - 1:].double())
    first = ops.mxfp8_quantize(x[:1])
    assert torch.equal(rows.codes[:T - 1].view(torch.uint8), first.codes.view(torch.uint8).expand(T - 1, n))
    assert torch.equal(ops.mxfp8_dequantize(rows)[T - 1:].double(), values8(last))


# ------------------------------------------------------------------ norms


def make(T, H, *, k=0, R=BF16, P=BF16, gate=None, post=True, pre=True, add_in=False, seed=1):
    n = lambda s, *shape: normal(*shape, seed=100 * seed + s)  # noqa: E731
    c = dict(resid=(2 * n(1, T, H)).to(R), post=(1 + 0.2 * n(2, H)).to(P) if post else None,
             pre=(1 + 0.2 * n(3, H)).to(P) if pre else None, k=k, add_in=None)
    shape = {None: None, "channel": (H,), "row": (1, H), "token": (T, 1), "full": (T, H)}[gate]
    c["gate"] = None if shape is None else n(4, *shape).to(P)
    if k:
        rows = T * k + 3
        c["y"] = n(5, rows, H).to(BF16)
        g = torch.Generator(device=DEV).manual_seed(seed)
        c["row_of"] = torch.randperm(rows, generator=g, device=DEV)[:T * k].to(torch.int32)
        c["w"] = torch.softmax(n(6, T, k), 1).to(BF16)
        c["add_in"] = n(7, T, H).to(BF16) if add_in else None
    else:
        c["block"] = n(8, T, H).to(BF16)
    return c


def call(c, **kw):
    args = dict(post_weight=c["post"], gate=c["gate"], pre_weight=c["pre"], want_mxfp8=True, **kw)
    if c["k"]:
        return ops.merge_norm_residual(c["y"], c["row_of"], c["w"], c["resid"], add_in=c["add_in"], **args)
    return ops.norm_residual(c["block"], c["resid"], **args)


def want64(c, scale=1.0, eps=1e-6):
    T, H = c["resid"].shape
    if c["k"]:
        at = c["row_of"].view(T, c["k"]).long()
        ok = (at >= 0) & (at < c["y"].shape[0])
        a = (c["y"].double()[at.clamp(0, c["y"].shape[0] - 1)] * (c["w"].double() * ok).unsqueeze(2)).sum(1)
        if c["add_in"] is not None:
            a = a + c["add_in"].double()
    else:
        a = c["block"].double()
    if c["post"] is not None:
        a = a / torch.sqrt(a.square().mean(1, keepdim=True) + eps) * c["post"].double()
    if c["gate"] is not None:
        a = a * c["gate"].double()
    # the scale is a float argument
    r = c["resid"].double() + float(torch.tensor(scale, dtype=F32)) * a
    eps = float(torch.tensor(eps, dtype=F32))
    n = r / torch.sqrt(r.square().mean(1, keepdim=True) + eps)
    return r, n if c["pre"] is None else n * c["pre"].double()


def check(c, got, scale=1.0, eps=1e-6):
    """64-bit sums of H + k terms are off by less than 2^-40: the sum and the norm are rounded once."""
    r, n = want64(c, scale, float(torch.tensor(eps, dtype=F32)))
    out_resid, out_norm, rows = got
    half = U if c["resid"].dtype is F32 else B
    if out_resid is not None:
        assert out_resid.dtype is c["resid"].dtype
        assert_within(out_resid, r, half * (1 + 2.0 ** -30) * r.abs() + 2.0 ** -38)
    if out_norm is not None:
        assert_within(out_norm, n, B * (1 + 2.0 ** -30) * n.abs() + 2.0 ** -38)
    same(rows, n)


@pytest.mark.parametrize("T,H", [(1, 32), (1, 2048), (2, 96), (5, 1504), (3, 4064), (2, 8192), (2, 8224), (3, 16384), (300, 2048)])
@pytest.mark.parametrize("gate,post,R,P", [(None, False, BF16, BF16), ("channel", True, F32, F32), ("token", False, BF16, F32),
                                           ("full", True, F32, BF16), ("row", False, F32, BF16)])
def test_norm(T, H, gate, post, R, P):
    c = make(T, H, R=R, P=P, gate=gate, post=post, seed=T)
    check(c, call(c, scale=0.75, eps=1e-5), 0.75, 1e-5)


@pytest.mark.parametrize("T,H,k", [(1, 2048, 8), (3, 64, 1), (17, 1504, 6), (130, 2048, 8), (2, 16384, 3)])
@pytest.mark.parametrize("post", [False, True])
def test_merge_and_norm(T, H, k, post):
    c = make(T, H, k=k, post=post, add_in=post, pre=not post, seed=k)
    c["row_of"][0], c["row_of"][-1] = -1, c["y"].shape[0]  # rows that are not there
    check(c, call(c))


def test_rows_at_addresses_that_16_bytes_do_not_divide():
    T, H = 3, 160
    c = make(T, H, seed=9)
    whole = call(c)
    for name in ("block", "resid"):
        room = torch.empty(T * H + 1, dtype=BF16, device=DEV)
        room[1:] = c[name].flatten()
        c[name] = room[1:].view(T, H)
    got = call(c)
    check(c, got)
    for a, b in zip(whole[:2], got[:2]):
        assert torch.equal(a, b)
    assert torch.equal(whole[2].codes.view(torch.uint8), got[2].codes.view(torch.uint8))
    codes = torch.empty(T * H + 4, dtype=torch.uint8, device=DEV)
    out = ops.MxRows(codes[4:].view(ops.F8).view(T, H), torch.empty((T, H // 32), dtype=torch.uint8, device=DEV))
    call(c, out_mxfp8=out)
    assert torch.equal(whole[2].codes.view(torch.uint8), out.codes.view(torch.uint8))


def test_outputs_given_left_out_and_in_place():
    c = make(40, 512, seed=3)
    r, n, rows = call(c)
    out = ops.mxfp8_empty(40, 512, DEV)
    got = call(c, want_resid=False, want_norm=False, out_mxfp8=out)
    assert got[0] is None and got[1] is None and got[2] is out
    assert torch.equal(out.codes.view(torch.uint8), rows.codes.view(torch.uint8)) and torch.equal(out.scales, rows.scales)
    resid, block = c["resid"].clone(), c["block"].clone()
    got = ops.norm_residual(block, resid, post_weight=c["post"], pre_weight=c["pre"], out_resid=resid, out_norm=block,
                            want_mxfp8=True)
    assert torch.equal(resid, r) and torch.equal(block, n)
    assert torch.equal(got[2].codes.view(torch.uint8), rows.codes.view(torch.uint8))


def test_norm_without_rows_is_as_before():
    """The call without 8-bit rows, which holds 32 bits, agrees with the one with them: its a is
    off by up to (H + 16) u |a| (a norm's sum, root and products, as in test_gpu_norm.py), and so is
    its r before the rounding, with |a| <= |r| + |resid|: where the two cancel, that is more than half
    a step of r.  Then both are rounded, to values of one step's distance where they differ.  The mean
    square and with it n is off by the same relative to the row, n's own by pre / rms."""
    c = make(50, 2048, seed=8)
    r0, n0 = ops.norm_residual(c["block"], c["resid"], post_weight=c["post"], pre_weight=c["pre"])
    r1, n1, _ = call(c)
    er = (2048 + 16) * U * (r1.double().abs() * (1 + B) + c["resid"].double().abs())
    assert_within(r0, r1.double(), 2.1 * B * r1.double().abs() + 1.1 * er)
    rms = r1.double().square().mean(1, keepdim=True).sqrt()
    en = 1.1 * er * c["pre"].double().abs() / rms + 2 * (2048 + 16) * U * n1.double().abs()
    assert_within(n0, n1.double(), 2.1 * B * n1.double().abs() + 1.1 * en)


def test_rows_with_infinities():
    c = make(4, 256, seed=6, post=False)
    c["resid"][1, 7], c["resid"][2, 100] = float("inf"), float("nan")
    _, n, rows = call(c)
    # an infinite sum of squares: the row's norm is 0, and NaN where the infinity was
    want = torch.zeros((4, 8), dtype=torch.bool, device=DEV)
    want[1, 0], want[2] = True, True
    assert torch.equal(rows.scales == 255, want)
    assert torch.equal(torch.isnan(values8(rows)).view(4, 8, 32).all(2), want)
    clean = make(4, 256, seed=6, post=False)
    _, _, plain = call(clean)
    for t in (0, 3):
        assert torch.equal(rows.codes[t].view(torch.uint8), plain.codes[t].view(torch.uint8))


def test_replay():
    c = make(16, 2048, k=4, seed=2)
    r, n, rows = [t.clone() if isinstance(t, torch.Tensor) else t for t in call(c)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(c)
    for _ in range(3):
        for t in (got[0], got[1], got[2].scales):
            t.zero_()
        got[2].codes.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], r) and torch.equal(got[1], n)
        assert torch.equal(got[2].codes.view(torch.uint8), rows.codes.view(torch.uint8))
        assert torch.equal(got[2].scales, rows.scales)


def test_refusals():
    x = normal(4, 64).to(BF16)
    with pytest.raises(ValueError, match="blocks of 32"):
        ops.mxfp8_quantize(normal(4, 48).to(BF16))
    with pytest.raises(ValueError, match="bfloat16"):
        ops.mxfp8_quantize(x.float())
    rows = ops.mxfp8_quantize(x)
    with pytest.raises(ValueError, match="codes must be"):
        ops.mxfp8_quantize(x[:3], out=rows)
    with pytest.raises(ValueError, match="scales must be"):
        ops.mxfp8_dequantize(ops.MxRows(rows.codes, rows.scales[:, :1].contiguous()))
    with pytest.raises(ValueError, match="MxRows"):
        ops.mxfp8_dequantize(x)
    with pytest.raises(ValueError, match="16-byte"):
        room = torch.empty(4 * 64 + 1, dtype=BF16, device=DEV)
        ops.mxfp8_quantize(room[1:].view(4, 64))
    with pytest.raises(ValueError, match="blocks of 32"):
        ops.norm_residual(normal(4, 40).to(BF16), normal(4, 40).to(BF16), want_mxfp8=True)
    with pytest.raises(ValueError, match="codes must be"):
        ops.norm_residual(x, x, out_mxfp8=ops.mxfp8_empty(4, 32, DEV))
