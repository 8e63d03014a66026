"""norm_residual and merge_norm_residual against their definition in 64 bits.

Bounds, with u = 2^-24 and half = half a step of the output's type: the merged sum is
off by (k + 2) u of its summed magnitudes; a norm multiplies that by (1 + (H + 8) u) at
most, relative to the value, and moves the mean square by the same; out_resid and out_norm
are rounded once.
"""
import pytest
import torch

from pdscope_amd import ops, stack

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def make(T, H, *, k=0, R=BF16, P=BF16, gate=None, post=True, pre=True, add_in=False, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    c = dict(resid=(2 * n(T, H)).to(R), post=(1 + 0.2 * n(H)).to(P) if post else None,
             pre=(1 + 0.2 * n(H)).to(P) if pre else None, k=k, add_in=None)
    shape = {None: None, "channel": (H,), "row": (1, H), "token": (T, 1), "full": (T, H)}[gate]
    c["gate"] = None if shape is None else n(*shape).to(P)
    if k:
        rows = T * k + 3
        c["y"] = n(rows, H).to(BF16)
        c["row_of"] = torch.randperm(rows, generator=g, device=DEV)[:T * k].to(torch.int32)
        c["w"] = torch.softmax(n(T, k), 1).to(BF16)
        c["add_in"] = n(T, H).to(BF16) if add_in else None
    else:
        c["block"] = n(T, H).to(BF16)
    return c


def call(c, **kw):
    args = dict(post_weight=c["post"], gate=c["gate"], pre_weight=c["pre"], **kw)
    if c["k"]:
        return ops.merge_norm_residual(c["y"], c["row_of"], c["w"], c["resid"], add_in=c["add_in"], **args)
    return ops.norm_residual(c["block"], c["resid"], **args)


def check(c, got, scale=1.0, eps=1e-6):
    resid = c["resid"].double()
    T, H = resid.shape
    if c["k"]:
        rows = c["row_of"].view(T, c["k"]).long()
        ok = (rows >= 0) & (rows < c["y"].shape[0])
        picked = c["y"].double()[rows.clamp(0, c["y"].shape[0] - 1)] * (c["w"].double() * ok).unsqueeze(2)
        a, mass = picked.sum(1), picked.abs().sum(1)
        if c["add_in"] is not None:
            a, mass = a + c["add_in"].double(), mass + c["add_in"].double().abs()
    else:
        a = c["block"].double()
        mass = a.abs()
    ea = (c["k"] + 2) * U * mass

    def rms(v, ev):
        """v / sqrt(mean(v^2) + eps), and its bound: the value's own error, and the
        mean's (2 |v| |ev| / H summed, H + 8 roundings) halved by the square root."""
        m = v.square().mean(1, keepdim=True) + eps
        em = (2 * (v.abs() * ev).mean(1, keepdim=True) + ev.square().mean(1, keepdim=True)) / m + (H + 8) * U
        return v / m.sqrt(), ev / m.sqrt() * (1 + em) + (v / m.sqrt()).abs() * em

    if c["post"] is not None:
        a, ea = rms(a, ea)
        a, ea = a * c["post"].double(), ea * c["post"].double().abs()
    g = 1.0 if c["gate"] is None else c["gate"].double()
    add = scale * g * a
    r = resid + add
    er = (abs(scale) * g * ea if c["gate"] is None else abs(scale) * g.abs() * ea) + 8 * U * (add.abs() + resid.abs())
    n, en = rms(r, er)
    if c["pre"] is not None:
        n, en = n * c["pre"].double(), en * c["pre"].double().abs()
    for t, want, e, dt in ((got[0], r, er, c["resid"].dtype), (got[1], n, en, BF16)):
        if t is None:
            continue
        half = torch.finfo(dt).eps / 2
        bound = e * (1 + half) + half * want.abs() + 4 * U * want.abs() + 2.0 ** -133
        assert t.dtype == dt and tuple(t.shape) == (T, H)
        off = (t.double() - want).abs()
        assert (off <= bound).all(), float((off / bound).max())


# H of one value, odd ones, one below and above a wave's and a workgroup's share, the largest
SIZES = [(1, 1), (3, 7), (1, 8), (2, 64), (5, 511), (4, 512), (3, 520), (2, 1000), (1, 2048), (33, 2048), (2, 3001),
         (1, 8192), (2, 8200), (2, 8191), (1, 16383), (1, 16384)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("R,P", [(BF16, BF16), (F32, F32)])
def test_norm_residual(T, H, R, P):
    c = make(T, H, R=R, P=P, gate="channel", seed=T + H)
    check(c, call(c, scale=0.5), 0.5)


@pytest.mark.parametrize("k", [1, 2, 6, 8, 17])
@pytest.mark.parametrize("T,H", [(1, 2048), (5, 130), (3, 2056), (70, 512)])
@pytest.mark.parametrize("R,P,add_in", [(F32, BF16, True), (BF16, F32, False)])
def test_merge_norm_residual(T, H, k, R, P, add_in):
    c = make(T, H, k=k, R=R, P=P, gate="token", add_in=add_in, seed=k + H)
    check(c, call(c))


@pytest.mark.parametrize("gate", [None, "channel", "row", "token", "full"])
@pytest.mark.parametrize("post,pre", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("T,H,k", [(4, 256, 0), (1, 77, 0), (4, 256, 3)])
def test_parts_that_may_be_left_out(gate, post, pre, T, H, k):
    c = make(T, H, k=k, gate=gate, post=post, pre=pre, P=F32, seed=2)
    check(c, call(c, scale=-1.5, eps=1e-3), -1.5, 1e-3)


def test_outputs_in_place_and_the_norm_alone():
    for H in (512, 77):
        c = make(6, H, gate="full", seed=4)
        want = call(c)
        r, n = call(c, want_resid=False)
        assert r is None and torch.equal(n, want[1])
        kept = dict(c, resid=c["resid"].clone())
        out = torch.empty_like(c["block"])
        r, n = call(c, out_resid=c["resid"], out_norm=out)
        assert r is c["resid"] and n is out
        assert torch.equal(r, want[0]) and torch.equal(n, want[1])
        r, n = call(kept, out_norm=kept["block"])  # over the block's output
        assert torch.equal(r, want[0]) and torch.equal(n, want[1])


@pytest.mark.parametrize("H", [1032, 2048, 10240])
def test_the_norm_over_its_own_input(H):
    """out_norm in the place of block or of resid, both rows read before they are written."""
    c = make(37, H)
    want = call(c)
    for name in ("block", "resid"):
        own = {**c, name: c[name].clone()}
        got = call(own, out_norm=own[name])
        assert got[1] is own[name]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_of_an_expert_computed_elsewhere_add_nothing():
    c = make(5, 256, k=4, seed=5)
    c["row_of"][[0, 7]] = -1
    c["row_of"][9] = c["y"].shape[0]
    c["row_of"][16:] = -1  # the last token has no row at all
    check(c, call(c))


def test_misaligned_rows_take_single_values():
    """Rows of 256 values at an odd element offset of their storage."""
    c = make(3, 256, seed=6)
    base = torch.zeros(3 * 256 + 1, dtype=BF16, device=DEV)
    base[1:] = c["block"].flatten()
    c["block"] = base[1:].view(3, 256)
    check(c, call(c))


def test_a_zero_row_and_a_row_with_nan():
    c = make(4, 300, seed=7)
    c["block"][1] = 0
    c["resid"][1] = 0
    want = [t.clone() for t in call(c)]
    assert torch.equal(want[1][1], torch.zeros_like(want[1][1]))
    c["block"][2, 5] = float("nan")
    got = call(c)
    for t, w in zip(got, want):
        assert torch.equal(t[[0, 1, 3]], w[[0, 1, 3]]) and torch.isnan(t[2]).all()


def test_equals_the_merge_that_it_replaces():
    """Without a norm and onto a zero residual, the sum is the layer's own merge."""
    c = make(64, 768, k=6, add_in=True, post=False, pre=False, seed=8)
    c["resid"].zero_()
    out = torch.empty((64, 768), dtype=BF16, device=DEV)
    ops.merge(c["y"], c["row_of"], c["w"], out, add_in=c["add_in"])
    r, _ = call(c)
    # two fp32 sums of seven values in another order, rounded once each
    step = (r.double() - out.double()).abs()
    assert (step <= 2 * 2.0 ** -8 * out.double().abs() + 16 * U * c["y"].abs().max()).all()
    assert (step != 0).double().mean() < 0.01


def test_replay_and_another_stream():
    c = make(9, 1024, k=4, R=F32, seed=9)
    want = call(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(c)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(c)
    for _ in range(3):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("k", [0, 1])
def test_rows_past_2_to_the_31_values(k):
    """1.1 million rows of 2048: the first, the last and some between have what a call over them
    alone gives."""
    T, H, n = 1_100_000, 2048, 1000
    g = torch.Generator(device=DEV).manual_seed(5)
    some = [torch.randn((n, H), generator=g, device=DEV).to(BF16) for _ in range(2)]
    block, resid = (t.repeat(T // n, 1) for t in some)
    block[-3:] = 2 * block[-3:]
    pre = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(BF16)
    if k:
        w = torch.ones((T, 1), dtype=BF16, device=DEV)
        got = ops.merge_norm_residual(block, torch.arange(T, dtype=torch.int32, device=DEV), w, resid, pre_weight=pre)
    else:
        got = ops.norm_residual(block, resid, pre_weight=pre)
    for rows in (slice(0, 7), slice(T // 2, T // 2 + 7), slice(T - 7, T)):
        want = ops.norm_residual(block[rows], resid[rows], pre_weight=pre)
        assert all(torch.equal(a[rows], b) for a, b in zip(got, want))


def test_refusals():
    c = make(4, 128)
    b, r = c["block"], c["resid"]
    for kw, match in ((dict(post_weight=c["post"], pre_weight=c["pre"].float()), "pre_weight must be"),
                      (dict(pre_weight=c["pre"][:64]), "pre_weight must be"),
                      (dict(gate=torch.ones(3, 128, dtype=BF16, device=DEV)), "gate must be"),
                      (dict(gate=torch.ones(4, dtype=BF16, device=DEV)), "gate must be"),
                      (dict(pre_weight=c["pre"].half()), "bf16 or fp32"),
                      (dict(out_norm=torch.empty(4, 128, device=DEV)), "out_norm"),
                      (dict(out_resid=torch.empty(4, 128, device=DEV)), "out_resid"),
                      (dict(eps=-1.0), "eps")):
        with pytest.raises(ValueError, match=match):
            ops.norm_residual(b, r, **kw)
    with pytest.raises(ValueError, match="resid must be"):
        ops.norm_residual(b, r[:3])
    with pytest.raises(ValueError, match="resid must be bf16 or fp32"):
        ops.norm_residual(b, r.half())
    with pytest.raises(ValueError, match="contiguous"):
        ops.norm_residual(b.t().contiguous().t(), r)
    with pytest.raises(ValueError, match="16384"):
        ops.norm_residual(torch.zeros(1, 16392, dtype=BF16, device=DEV), torch.zeros(1, 16392, dtype=BF16, device=DEV))
    with pytest.raises(ValueError, match="T >= 1"):
        ops.norm_residual(b[:0], r[:0])
    m = make(4, 128, k=2)
    with pytest.raises(ValueError, match="row_of"):
        ops.merge_norm_residual(m["y"], m["row_of"][:7], m["w"], m["resid"])
    with pytest.raises(ValueError, match="rows of 128"):
        ops.merge_norm_residual(m["y"].flatten()[:-1], m["row_of"], m["w"], m["resid"])
    with pytest.raises(ValueError, match="add_in"):
        ops.merge_norm_residual(m["y"], m["row_of"], m["w"], m["resid"], add_in=m["resid"][:2])


def test_stack_with_the_fused_norm():
    """Every block's input in a session with fused_norm is the norm of the block
    before: the sum and its norm in 64 bits, within (H + 8) / 2 + 4 roundings of fp32
    and the one to bf16."""
    model = stack.build_stack(3, torch.device(DEV, 0), hot_per_layer=6, calib_tokens=64, H=512, I=256, E=32, k=4)
    session = stack.StackSession(model, torch.device(DEV, 0), stack.StackBudget(demand_slots=4), fused_norm=True)
    try:
        for step, T in enumerate((5, 1)):
            calls = []
            x = torch.randn(T, model.H, device=DEV, generator=torch.Generator(DEV).manual_seed(step)).to(BF16)
            last, _ = session.run_pass(x, step, lambda c: calls.append((c.x.clone(), c.out.clone())))
            torch.cuda.synchronize()
            assert torch.equal(calls[0][0], x)
            for (xin, out), got in zip(calls, [c[0] for c in calls[1:]] + [last]):
                h = xin.double() + out.double()
                want = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6)
                bound = want.abs() * (((model.H + 8) / 2 + 4) * U + 2.0 ** -8) + 2.0 ** -133
                assert ((got.double() - want).abs() <= bound).all()
    finally:
        session.close()
