"""The layer of 1 to 16 tokens (ops.moe_few, layer.moe_few) over bf16 and 4-bit experts
against its definition in 64 bits."""
import pytest
import torch

from moe64 import assert_within, merged64, routed64
from pdscope_amd import layer, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Layer:
    def __init__(self, T, H, I, E, k, rep, *, seed=1, bias=None, add_in=False, ws=None, spread=0.02):
        g = torch.Generator(device=DEV).manual_seed(seed)
        n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
        self.T, self.H, self.I, self.E, self.k, self.rep = T, H, I, E, k, rep
        self.x = n(T, H).to(torch.bfloat16)
        self.gate = (spread * n(E, H)).to(torch.bfloat16)
        self.experts = (0.05 * n(E, 3 * I * H)).to(torch.bfloat16)
        if rep == "mxfp4":
            self.blocks = ops.mxfp4_quantize(self.experts, H, I)
            self.experts = ops.mxfp4_dequantize(self.blocks, H, I)
        else:
            self.blocks = self.experts
        self.slots = ops.slot_table([self.blocks[e] for e in range(E)], DEV)
        self.bias = n(E) if bias else None
        self.add_in = n(T, H).to(torch.bfloat16) if add_in else None
        self.ws = ws or layer.MoEWorkspace(T, H, I, E, k, DEV, few_tokens=True)

    def run(self, normalize=True):
        return layer.moe_few(self.x, self.gate, self.slots, self.ws, normalize=normalize, bias=self.bias,
                             add_in=self.add_in, representation=self.rep)

    def block_of(self, e):
        return self.experts[e].double() if int(self.slots[e]) else None

    def check(self, got, normalize=True):
        out, logits, ids, w = got
        x = self.x.double()
        want_logits, want_ids, want_w = routed64(x, self.gate.double(), self.bias, self.k, normalize)
        assert torch.equal(logits, want_logits)
        assert torch.equal(ids.long(), want_ids)
        # fp32 exp and sums, one rounding to bf16
        assert_within(w, want_w, (2.0 ** -8 + 2.0 ** -18) * want_w)
        want, bound = merged64(x, ids.long(), w.double(), self.block_of, self.H, self.I,
                               None if self.add_in is None else self.add_in.double())
        assert_within(out, want, bound)


# the smallest shapes, odd token counts, experts off every power of two, groups of H that
# do not deal evenly to eight waves (384, 1152, 1536, 2176), more experts than a wave
SHAPES = [(1, 128, 128, 1, 1), (16, 128, 128, 1, 1), (2, 128, 128, 3, 3), (3, 256, 128, 5, 2), (5, 384, 256, 8, 4),
          (7, 512, 384, 60, 6), (1, 1024, 512, 64, 4), (11, 1024, 512, 64, 4), (16, 1152, 128, 96, 16),
          (9, 1536, 384, 96, 6), (1, 2048, 768, 128, 8), (2, 2048, 768, 128, 8), (16, 2048, 768, 128, 8),
          (15, 2048, 256, 256, 8), (16, 2048, 1408, 64, 6), (4, 2176, 128, 40, 3), (13, 3200, 256, 16, 2),
          (6, 4096, 256, 12, 5)]


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
@pytest.mark.parametrize("T,H,I,E,k", SHAPES)
def test_layer(T, H, I, E, k, rep):
    lay = Layer(T, H, I, E, k, rep, seed=T + H + E)
    lay.check(lay.run())


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
@pytest.mark.parametrize("T,normalize", [(1, False), (4, True), (16, False)])
def test_bias_add_in_and_unnormalised_weights(T, normalize, rep):
    lay = Layer(T, 512, 256, 48, 5, rep, bias=True, add_in=True, seed=7)
    lay.check(lay.run(normalize), normalize)


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
def test_equal_logits_take_the_lower_expert(rep):
    lay = Layer(6, 256, 128, 24, 6, rep, seed=3)
    lay.gate[1::2] = lay.gate[0::2]  # every logit twice
    lay.gate[20:] = 0
    lay.check(lay.run())


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
def test_every_token_on_the_same_experts(rep):
    """The list is k experts long whatever T: many pieces per expert, 16 rows each."""
    lay = Layer(16, 512, 768, 32, 2, rep, bias=True, seed=4)
    lay.bias[:] = 0
    lay.bias[[9, 30]] = 50.0
    lay.check(lay.run())


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
@pytest.mark.parametrize("T", [1, 13])
def test_experts_without_a_copy_add_nothing(rep, T):
    lay = Layer(T, 384, 256, 16, 4, rep, add_in=True, seed=5)
    lay.slots[::2] = 0
    lay.check(lay.run())
    lay.slots[:] = 0
    out, _, _, _ = lay.run()
    assert torch.equal(out, lay.add_in)
    lay.add_in = None
    out, _, _, _ = lay.run()
    assert torch.equal(out, torch.zeros_like(out))


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
@pytest.mark.parametrize("E,k", [(8, 2), (40, 9), (128, 8)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_token_with_nan_keeps_to_itself(rep, E, k, bad):
    lay = Layer(5, 256, 128, E, k, rep, seed=6)
    clean = [t.clone() for t in lay.run()]
    lay.x[3, 17] = bad
    out, logits, ids, w = lay.run()
    rest = [0, 1, 2, 4]
    for got, want in zip((logits, ids, w), clean[1:]):
        assert torch.equal(got[rest], want[rest])
    assert torch.isfinite(out[rest].float()).all() and not torch.isfinite(out[3].float()).any()
    assert ids.min() >= 0 and ids.max() < E and ids[3].unique().numel() == k


def test_replays_other_streams_and_a_larger_workspace():
    """One workspace for up to 16 tokens serves smaller batches; a captured call replays to
    the eager result, with eager work of another batch on the same workspace in between."""
    lay = Layer(16, 512, 256, 32, 4, "mxfp4", seed=8)
    few = Layer(3, 512, 256, 32, 4, "mxfp4", seed=9, ws=lay.ws)
    want = [t.clone() for t in lay.run()]
    few.check(few.run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lay.run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = lay.run()
    for _ in range(4):
        for t in got:
            t.zero_()
        few.run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = lay.x.clone()
    lay.x.copy_(x.flip(0))  # the captured call reads its inputs anew
    graph.replay()
    torch.cuda.synchronize()
    lay.check([t.clone() for t in got])


def test_the_same_call_gives_the_same_bits():
    for rep in ("mxfp4", "bf16"):
        lay = Layer(12, 1024, 512, 64, 6, rep, seed=10)
        want = [t.clone() for t in lay.run()]
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(lay.run(), want))


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
@pytest.mark.parametrize("masked", [float("-inf"), torch.finfo(torch.float32).min])
@pytest.mark.parametrize("T,E,k,left", [(1, 32, 4, 5), (5, 160, 4, 4), (16, 96, 6, 3), (2, 8, 8, 1)])
@pytest.mark.parametrize("normalize", [True, False])
def test_a_bias_that_masks_experts(T, E, k, left, masked, normalize, rep):
    """All but `left` experts masked, in one case fewer than k: masked ones are then picked by
    ascending id, with weight 0."""
    lay = Layer(T, 256, 128, E, k, rep, bias=True, seed=12)
    keep = torch.randperm(E, generator=torch.Generator().manual_seed(13))[:left].to(DEV)
    bias = torch.full((E,), masked, device=DEV)
    bias[keep] = lay.bias[keep]
    lay.bias = bias
    got = lay.run(normalize)
    lay.check(got, normalize)
    assert torch.isin(got[2][:, :min(k, left)].long(), keep).all() and not got[3][:, left:].any()


def test_two_calls_at_once_and_graphs_that_share_a_workspace():
    """Two streams with a workspace each; then two captured calls of different sizes on one
    workspace, replayed in turn."""
    a, b = Layer(16, 1024, 256, 64, 6, "mxfp4", seed=14), Layer(7, 1024, 512, 64, 4, "bf16", seed=15)
    want = [[t.clone() for t in lay.run()] for lay in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for lay, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                lay.run()
    torch.cuda.synchronize()
    for lay, w in zip((a, b), want):
        assert torch.equal(lay.ws.out[:lay.T], w[0]) and torch.equal(lay.ws.ids[:lay.T], w[2])

    ws = torch.empty(max(lay.ws.few_ws.numel() for lay in (a, b)), dtype=torch.uint8, device=DEV)
    graphs, outs = [], []
    for lay, w in zip((a, b), want):
        o = [torch.empty_like(t) for t in w]

        def call(lay=lay, o=o):
            ops.moe_few(lay.x, lay.gate, lay.slots, lay.I, lay.k, True, representation=lay.rep, out=o[0], logits=o[1],
                        ids=o[2], weights=o[3], workspace=ws)

        call()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call()
        outs.append(o)
    for _ in range(4):
        for g, o, w in zip(graphs, outs, want):
            for t in o:
                t.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(t, v) for t, v in zip(o, w))


@pytest.mark.parametrize("T", [1, 7, 16])
@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
def test_the_layer_over_its_own_output(rep, T):
    """A step whose activations (and the shared experts' sum) lie where the layer's
    output goes, as a stack that keeps one buffer has it."""
    lay = Layer(T, 512, 256, 16, 4, rep)
    want = [t.clone() for t in layer.moe_few(lay.x, lay.gate, lay.slots, lay.ws, add_in=lay.x, representation=rep)]
    x = lay.ws.out[:T]
    x.copy_(lay.x)
    got = layer.moe_few(x, lay.gate, lay.slots, lay.ws, add_in=x, representation=rep)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
def test_the_largest_layer(rep):
    """Every limit but that on I at once: 16 tokens, 256 experts (eight blocks, each in 32 slots), k = 16 and
    H = 4096, with more partial rows than 16 bits count."""
    T, H, I, E, k = 16, 4096, 8320, 256, 16
    lay = Layer(T, H, I, 8, 8, rep, seed=16)
    g = torch.Generator(device=DEV).manual_seed(17)
    lay.E, lay.k = E, k
    lay.gate = (0.02 * torch.randn((E, H), generator=g, device=DEV)).to(torch.bfloat16)
    lay.slots = lay.slots.repeat(E // 8)
    lay.ws = layer.MoEWorkspace(T, H, I, E, k, DEV, few_tokens=True)
    lay.block_of = lambda e: lay.experts[e % 8].double()
    lay.check(lay.run())


def test_refusals():
    lay = Layer(4, 256, 128, 8, 2, "bf16")
    x17 = torch.zeros((17, 256), dtype=torch.bfloat16, device=DEV)
    ws17 = layer.MoEWorkspace(17, 256, 128, 8, 2, DEV, few_tokens=True)
    with pytest.raises(ValueError, match="unsupported shape T=17"):
        layer.moe_few(x17, lay.gate, lay.slots, ws17)
    with pytest.raises(ValueError, match="few_tokens=True"):
        layer.moe_few(lay.x, lay.gate, lay.slots, layer.MoEWorkspace(4, 256, 128, 8, 2, DEV))
    with pytest.raises(ValueError, match="outside moe_few"):
        layer.MoEWorkspace(4, 256, 192, 8, 2, DEV, few_tokens=True)
    with pytest.raises(ValueError, match="representation"):
        layer.moe_few(lay.x, lay.gate, lay.slots, lay.ws, representation="int4")
    with pytest.raises(ValueError, match="router input"):
        layer.moe_few(lay.x[:, :128].contiguous(), lay.gate, lay.slots, lay.ws)
    with pytest.raises(ValueError, match="bias"):
        layer.moe_few(lay.x, lay.gate, lay.slots, lay.ws, bias=torch.zeros(7, device=DEV))
    with pytest.raises(ValueError, match="add_in"):
        layer.moe_few(lay.x, lay.gate, lay.slots, lay.ws, add_in=lay.x[:3])
    with pytest.raises(ValueError, match="slots"):
        layer.moe_few(lay.x, lay.gate, lay.slots[:5], lay.ws)
    with pytest.raises(ValueError, match="contiguous"):
        layer.moe_few(lay.x.t().contiguous().t(), lay.gate, lay.slots, lay.ws)
    with pytest.raises(ValueError, match="workspace too small"):
        out, logits, ids, w = lay.run()
        ops.moe_few(lay.x, lay.gate, lay.slots, 128, 2, True, out=out, logits=logits, ids=ids, weights=w,
                    workspace=lay.ws.few_ws[:256])
