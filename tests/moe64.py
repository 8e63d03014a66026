"""The MoE layer in 64 bits with, beside every value, how far a kernel may be off it.

The kernels under test hold sums in fp32 and round h to bf16 (and, in the prompt
form, each expert's row); with u = 2^-24 and b = 2^-8 (half a step of bf16):
  gate, up       (H + 2) u (|x| . |w|)
  h = silu(g) u  the above through |silu'| <= 1.1, 2^-20 |h| for the hardware's
                 exp2 and reciprocal, b |h| for its rounding
  down           |d| . (error of h) + (I + 2) u (|d| . |h|), b |y| where rows are rounded
  out            sum of w times that, (n + 2) u of the summed magnitudes, b |out|
"""
import torch

U, B = 2.0 ** -24, 2.0 ** -8


def expert64(block, x, H, I, rounded_rows):
    """(y, bound) of x [n, H] through one expert block [3IH], all fp64."""
    g_w, u_w, d_w = block[:I * H].view(I, H), block[I * H:2 * I * H].view(I, H), block[2 * I * H:].view(H, I)
    g, u = x @ g_w.T, x @ u_w.T
    eg, eu = ((H + 2) * U * (x.abs() @ w.abs().T) for w in (g_w, u_w))
    s = g * torch.sigmoid(g)
    h = s * u
    eh = (1 + B) * (1.1 * eg * u.abs() + s.abs() * eu + 1.1 * eg * eu) + (B + 2.0 ** -20) * h.abs() + 2.0 ** -133
    y = h @ d_w.T
    ey = eh @ d_w.abs().T + (I + 2) * U * ((h.abs() + eh) @ d_w.abs().T)
    if rounded_rows:
        ey = ey * (1 + B) + B * y.abs() + 2.0 ** -133
    return y, ey


def merged64(x, ids, w, block_of, H, I, add_in=None, rounded_rows=False):
    """(out, bound) of the routed experts' weighted sum for a given routing; block_of(e)
    is expert e's fp64 block or None (no copy: adds nothing)."""
    out = torch.zeros((x.shape[0], H), dtype=torch.float64, device=x.device)
    bound, mass = torch.zeros_like(out), torch.zeros_like(out)
    for e in torch.unique(ids).tolist():
        block = block_of(e)
        if block is None:
            continue
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        y, ey = expert64(block, x[t], H, I, rounded_rows)
        ws = w[t, slot].unsqueeze(1)
        out.index_add_(0, t, ws * y)
        bound.index_add_(0, t, ws * ey)
        mass.index_add_(0, t, ws * (y.abs() + ey))
    if add_in is not None:
        out += add_in
        mass += add_in.abs()
    # up to k I / 32 partial rows a token, and as many products with w
    bound += (ids.shape[1] * (I // 32) + 4) * U * mass
    return out, bound * (1 + B) + B * out.abs() + 2.0 ** -133


def routed64(x, gate, bias, k, normalize):
    """(logits bf16, ids, weights fp64): logits are bf16 by definition, and the selection
    is made on them."""
    logits = (x @ gate.T).to(torch.bfloat16)
    seen = logits.double() if bias is None else (logits.float() + bias.float()).double()
    p = torch.softmax(seen, dim=1)
    ids = torch.sort(seen, dim=1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    return logits, ids, w / w.sum(1, keepdim=True) if normalize else w


def assert_within(got, want, bound):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off; worst {float((off / bound).nan_to_num(9e9).max()):.3g} "
                           f"of the bound at {torch.nonzero(bad)[0].tolist()}")
