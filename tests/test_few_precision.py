"""What the layer of 1 to 16 tokens keeps of h and of the experts' rows, which its own rounding
of the output hides elsewhere.

Tokens of few values that are not 0, down rows of few weights that are not 0 (zeros add
exactly, so that every sum is short) and a summand that takes away all of the output but its last
bits: then a value is off by little more than what the kernel drops of h.  With u = 2^-24,
N values of a token and M weights of a down row:
  gate, up   2 N u (|x| . |w|): the matrix cores may cut off where they add
  h          the above through |silu'| <= 1.1, 2^-20 |h| for the hardware's exp2 and
             reciprocal and the product's rounding, and what two bf16 parts drop of it: the
             first is cut off (the rest is below 2^-7 of h's power of two), the second is
             half a step of 8 bits off: 2^-16 |h|, and 2^-23 |h| where a rest of 0 is made 2^-24 h
  rows       |d| . (error of h) + 2 (2 M + 2) u (|d| . |h|): two products a weight
  out        sum of w times that, (k M + 4) u of the summed magnitudes (a partial row has
             at least one weight, each is multiplied by w), 2^-8 |out|
A single bf16 h would be up to 2^-8 |h| off.
"""
import pytest
import torch

from pdscope_amd import layer, ops

BF16 = torch.bfloat16
U, B, N, M = 2.0 ** -24, 2.0 ** -8, 8, 4
TWO_PARTS = 2.0 ** -16 + 2.0 ** -23


class Case:
    def __init__(self, T, H, I, E, k, rep, device, seed):
        g = torch.Generator().manual_seed(seed)
        n = lambda *s: torch.randn(s, generator=g)  # noqa: E731

        def few(rows, cols, count):
            """Rows of `count` values that are not 0, at places of their own."""
            at = torch.rand((rows, cols), generator=g).topk(count, dim=1).indices
            return torch.zeros((rows, cols)).scatter_(1, at, n(rows, count))

        self.T, self.H, self.I, self.E, self.k, self.rep = T, H, I, E, k, rep
        self.x = few(T, H, N).to(BF16).to(device)
        self.gate = n(E, H).to(BF16).to(device)
        self.experts = torch.empty((E, 3 * I * H), dtype=BF16, device=device)
        for e in range(E):
            self.experts[e, :2 * I * H] = (0.5 * n(2 * I * H)).to(BF16)
            self.experts[e, 2 * I * H:] = few(H, I, M).to(BF16).flatten()
        if rep == "mxfp4":
            self.blocks = ops.mxfp4_quantize(self.experts, H, I)
            self.experts = ops.mxfp4_dequantize(self.blocks, H, I)
        else:
            self.blocks = self.experts

    def want(self, ids, w, add_in=None):
        """(out, bound, per expert (tokens, slots, h, down matrix)), in 64 bits, for a routing."""
        T, H, I, k = self.T, self.H, self.I, self.k
        x, w = self.x.double(), w.double()
        out = torch.zeros((T, H), dtype=torch.float64, device=x.device)
        err, mass, parts = torch.zeros_like(out), torch.zeros_like(out), []
        for e in torch.unique(ids).tolist():
            t, slot = torch.nonzero(ids == e, as_tuple=True)
            g_w, u_w, d_w = (m.double() for m in self.experts[e].split(I * H))
            g_w, u_w, d_w = g_w.view(I, H), u_w.view(I, H), d_w.view(H, I)
            g, u = x[t] @ g_w.T, x[t] @ u_w.T
            eg, eu = (2 * N * U * (x[t].abs() @ m.abs().T) for m in (g_w, u_w))
            s = g * torch.sigmoid(g)
            h = s * u
            eh = 1.1 * eg * u.abs() + s.abs() * eu + 1.1 * eg * eu + (2.0 ** -20 + TWO_PARTS) * h.abs() + 2.0 ** -133
            y, ay = h @ d_w.T, (h.abs() + eh) @ d_w.abs().T
            ey = eh @ d_w.abs().T + 2 * (2 * M + 2) * U * ay
            ws = w[t, slot].unsqueeze(1)
            out.index_add_(0, t, ws * y)
            err.index_add_(0, t, ws * ey)
            mass.index_add_(0, t, ws * ay)
            parts.append((t, ws, h, d_w))
        if add_in is not None:
            out = out + add_in.double()
            mass = mass + add_in.double().abs()
        err = err + (k * M + 4) * U * mass
        return out, err * (1 + B) + B * out.abs() + 2.0 ** -133, parts

    def last_bits(self, ids, w):
        """The summand, and what is left of the output with it."""
        add_in = -self.want(ids, w)[0].to(BF16)
        return (add_in, *self.want(ids, w, add_in))


def two_parts(h):
    h = h.float()
    first = (h.view(torch.int32) & -65536).view(torch.float32)
    return first.double(), (h - first).to(BF16).double()


KEPT = {
    "two parts": lambda h: sum(two_parts(h)),
    "one part": lambda h: h.to(BF16).double(),
    "one part, cut off": lambda h: two_parts(h)[0],
    "the rest twice": lambda h: two_parts(h)[0] + 2 * two_parts(h)[1],
    "the rest of another column": lambda h: two_parts(h)[0] + two_parts(h)[1].roll(1, 1),
    "the rest of another half": lambda h: two_parts(h)[0] + two_parts(h)[1].roll(16, 1),
    "the rest of another token": lambda h: two_parts(h)[0] + two_parts(h)[1].roll(1, 0),
}


@pytest.mark.parametrize("kept", KEPT)
@pytest.mark.parametrize("T,H,I,E,k", [(5, 128, 128, 4, 4), (16, 256, 256, 6, 3)])
def test_the_bound_tells_them_apart(T, H, I, E, k, kept):
    """On the CPU: two parts of h are within the bound everywhere; with any of the mistakes a
    third of the values at least are beyond it."""
    c = Case(T, H, I, E, k, "bf16", "cpu", seed=T)
    logits = (c.x.double() @ c.gate.double().T).to(BF16).double()
    w, ids = torch.softmax(logits, 1).topk(k, dim=1)
    w = w.to(BF16)
    add_in, want, bound, parts = c.last_bits(ids, w)
    out = add_in.double()
    for t, ws, h, d_w in parts:
        # the rest of another token is 0 where an expert has only one
        out = out.index_add(0, t, ws * (KEPT[kept](h) @ d_w.T))
    off = (out.float().to(BF16).double() - want).abs() > bound
    if kept == "two parts":
        assert not off.any()
    else:
        assert off.double().mean() > 1 / 3


# from the smallest layer to the framework's own; activations in registers and in LDS, groups
# of H that do not deal evenly to eight waves
@pytest.mark.gpu
@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
@pytest.mark.parametrize("T,H,I,E,k", [(1, 128, 128, 1, 1), (16, 128, 128, 4, 2), (3, 384, 256, 8, 4), (7, 1024, 512, 16, 4),
                                       (16, 1536, 384, 12, 6), (1, 2048, 768, 12, 8), (5, 2048, 768, 12, 8),
                                       (16, 2048, 1408, 8, 6), (9, 2176, 128, 12, 3), (16, 3200, 256, 8, 2),
                                       (6, 4096, 256, 12, 5)])
def test_what_the_kernel_keeps(T, H, I, E, k, rep):
    c = Case(T, H, I, E, k, rep, "cuda", seed=T + H)
    slots = ops.slot_table([c.blocks[e] for e in range(E)], "cuda")
    ws = layer.MoEWorkspace(T, H, I, E, k, "cuda", few_tokens=True)
    _, _, ids, w = (t.clone() for t in layer.moe_few(c.x, c.gate, slots, ws, representation=rep))
    add_in, want, bound, _ = c.last_bits(ids, w)
    out, _, ids2, w2 = layer.moe_few(c.x, c.gate, slots, ws, add_in=add_in, representation=rep)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    off = (out.double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16])
def test_the_layer_of_four_bit_experts(T):
    """moe_forward's own way for so few tokens, with the summand as shared experts would add it."""
    H, I, E, k = 512, 256, 32, 4
    c = Case(T, H, I, E, k, "mxfp4", "cuda", seed=T)
    slots = ops.slot_table([c.blocks[e] for e in range(E)], "cuda")
    ws = layer.MoEWorkspace(T, H, I, E, k, "cuda", few_tokens=True)
    out, _, ids, w = layer.moe_forward(c.x, c.gate, slots, ws, representation="mxfp4")
    want, bound, _ = c.want(ids, w)
    assert ((out.double() - want).abs() <= bound).all()
