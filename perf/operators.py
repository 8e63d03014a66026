"""Operators of the MoE-layer path over 4-bit experts and small batches.

Four operators, used together by a serving step of a stack of MoE blocks:

* ``quantize``: bf16 expert blocks to microscaled 4-bit floating point
  (e2m1 values, one e8m0 scale per 32 consecutive inputs of a row) and back;
* ``few``: the whole MoE layer (router, selection, SwiGLU experts, weighted
  merge) of 1 to 16 tokens, over bf16 or 4-bit experts;
* ``grouped``: the routed SwiGLU experts of a prompt over 4-bit experts;
* ``norm``: the norm after a block, its gate and residual scale, the residual
  sum and the norm before the next block, on a block's output or on the
  experts' rows that the MoE merge would sum first.

Weights are N(0, 0.02), activations N(0, 1), as in the framework's synthetic
layers; 4-bit weights are those weights quantised.  A state keeps them as a
checkpoint does, as packed codes and scales in row-major order; a program of
the framework also keeps the expert blocks laid out from them, its slot table
and its workspaces.
"""
import math

import torch

own = False
DEV = "cuda"
BF16 = torch.bfloat16

SHAPES = {
    # the two layer shapes of pdscope_amd.synthetic (dsv2: its always-on shared
    # experts' output is added to the routed experts' sum)
    "qwen": dict(H=2048, I=768, E=128, k=8, normalize=True, add_in=False),
    "dsv2": dict(H=2048, I=1408, E=64, k=6, normalize=False, add_in=True),
    # smaller layers: fewer experts, a narrower hidden size
    "small": dict(H=1024, I=512, E=64, k=4, normalize=True, add_in=False),
    "narrow": dict(H=1536, I=384, E=96, k=6, normalize=True, add_in=False),
}
FEW = 16


def listed():
    return [
        # one expert on its way into a device copy: what staging a missing expert adds
        dict(name="quantize_qwen_e1", op="quantize", shape="qwen", E=1),
        # every expert of a layer, when a model is loaded
        dict(name="quantize_dsv2_e64", op="quantize", shape="dsv2", E=64),
        # the decode step of one user through 8 layers of 4-bit experts: latency
        dict(name="few_qwen_4bit_t1", op="few", shape="qwen", rep="mxfp4", T=1, layers=8, bias=False),
        # a few requests at once, each with experts of its own
        dict(name="few_qwen_4bit_t5", op="few", shape="qwen", rep="mxfp4", T=5, layers=4, bias=True),
        # a full small batch (or the drafted tokens of a few requests) with shared experts
        dict(name="few_dsv2_4bit_t16", op="few", shape="dsv2", rep="mxfp4", T=16, layers=2, bias=False),
        # two requests over bf16 experts
        dict(name="few_qwen_bf16_t2", op="few", shape="qwen", rep="bf16", T=2, layers=4, bias=False),
        # an odd number of them through the small layer
        dict(name="few_small_bf16_t11", op="few", shape="small", rep="bf16", T=11, layers=4, bias=False),
        # a batch just too large for the few-token form: one or two rows an expert
        dict(name="grouped_qwen_t33", op="grouped", shape="qwen", T=33, skew=False),
        # a mixed batch of decode tokens and prompt chunks, an odd length, uneven routing
        dict(name="grouped_dsv2_t1303", op="grouped", shape="dsv2", T=1303, skew=True),
        # a long prompt
        dict(name="grouped_qwen_t4096", op="grouped", shape="qwen", T=4096, skew=False),
        # between two blocks, one token: latency
        dict(name="norm_t1", op="norm", T=1, H=2048, k=0, resid="bf16", params="bf16", gate="none", post=False),
        # after the experts of a long prompt, the merge of 8 rows a token included
        dict(name="norm_merge_t4096", op="norm", T=4096, H=2048, k=8, resid="fp32", params="bf16", gate="channel",
             post=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "few", "few", "few", "grouped", "grouped", "norm", "norm"])
    if op == "quantize":
        shape = rng.choice(sorted(SHAPES))
        return dict(op=op, shape=shape, E=_log_int(rng, 1, 64))
    if op == "few":
        return dict(op=op, shape=rng.choice(sorted(SHAPES)), rep=rng.choice(["mxfp4", "mxfp4", "bf16"]),
                    T=rng.randint(1, FEW), layers=rng.randint(1, 2), bias=rng.random() < 0.5)
    if op == "grouped":
        return dict(op=op, shape=rng.choice(sorted(SHAPES)), T=_log_int(rng, FEW + 1, 4095), skew=rng.random() < 0.5)
    return dict(op=op, T=_log_int(rng, 1, 4095), H=rng.choice([rng.randint(64, 4095), 8 * rng.randint(8, 512), 2048]),
                k=rng.choice([0, 0, 1, 4, 6, 8]), resid=rng.choice(["bf16", "fp32"]),
                params=rng.choice(["bf16", "fp32"]), gate=rng.choice(["none", "channel", "token", "full"]),
                post=rng.random() < 0.6)


# ------------------------------------------------------------------ inputs


def _normal(gen, shape, std=1.0, dtype=BF16):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * std).to(dtype)


def _quantize(w):
    """Codes [.., K/2] and scales [.., K/32] of w [.., K]: the block's scale is
    2^(floor(log2 of its largest magnitude) - 2), so that it lies in [4, 8); each
    value is rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the
    even code, above 6 to 6).  Value 2i of a row in the low half of byte i."""
    b = w.float().unflatten(-1, (-1, 32))
    s = (torch.frexp(b.abs().amax(-1)).exponent - 3).clamp(-127, 127)
    s = torch.where(b.abs().amax(-1) > 0, s, -127)
    a = torch.ldexp(b, -s.unsqueeze(-1))
    m = a.abs()
    code = torch.where(m < 2, torch.round(2 * m), torch.where(m < 4, torch.round(m) + 2, torch.round(m / 2) + 4))
    code = (code.clamp(max=7) + 8 * torch.signbit(a)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (s + 127).to(torch.uint8)


def _checkpoint(gen, E, numel, block=1 << 25):
    """4-bit weights of E experts of `numel` values: N(0, 0.02) quantised."""
    codes = torch.empty((E, numel // 2), dtype=torch.uint8, device=DEV)
    scales = torch.empty((E, numel // 32), dtype=torch.uint8, device=DEV)
    step = max(1, block // numel)
    for e in range(0, E, step):
        n = min(step, E - e)
        codes[e:e + n], scales[e:e + n] = _quantize(_normal(gen, (n, numel), 0.02))
    return codes, scales


def _weights(gen, E, numel, block=1 << 25):
    out = torch.empty((E, numel), dtype=BF16, device=DEV)
    step = max(1, block // numel)
    for e in range(0, E, step):
        out[e:e + step] = _normal(gen, (min(step, E - e), numel), 0.02)
    return out


class _Few:
    def __init__(self, case, gen):
        s = SHAPES[case["shape"]]
        H, I, E, T = s["H"], s["I"], s["E"], case["T"]
        self.rep, self.k, self.normalize, self.H, self.I = case["rep"], s["k"], s["normalize"], H, I
        self.layers = []
        for _ in range(case["layers"]):
            lay = dict(gate=_normal(gen, (E, H), 0.02), x=_normal(gen, (T, H)))
            lay["bias"] = torch.randn(E, generator=gen, device=DEV) * 0.5 if case["bias"] else None
            lay["add_in"] = _normal(gen, (T, H), 0.5) if s["add_in"] else None
            if self.rep == "mxfp4":
                lay["codes"], lay["scales"] = _checkpoint(gen, E, 3 * I * H)
            else:
                lay["experts"] = _weights(gen, E, 3 * I * H)
            self.layers.append(lay)
        self.graph = None
        if own:
            from pdscope_amd import layer, ops
            for lay in self.layers:
                if self.rep == "mxfp4":
                    lay["experts"] = ops.mxfp4_pack(lay["codes"], lay["scales"], H, I)
                lay["slots"] = ops.slot_table([lay["experts"][e] for e in range(E)], DEV)
                lay["ws"] = layer.MoEWorkspace(T, H, I, E, s["k"], DEV, few_tokens=True)
            # a serving loop captures its decode step once and replays it
            cur, side = torch.cuda.current_stream(), torch.cuda.Stream()
            side.wait_stream(cur)
            with torch.cuda.stream(side):
                self.step()
            cur.wait_stream(side)
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.outputs = self.step()

    def step(self):
        from pdscope_amd import layer
        return [layer.moe_few(lay["x"], lay["gate"], lay["slots"], lay["ws"], normalize=self.normalize,
                              bias=lay["bias"], add_in=lay["add_in"], representation=self.rep)
                for lay in self.layers]


class _Grouped:
    def __init__(self, case, gen):
        s = SHAPES[case["shape"]]
        H, I, E, k, T = s["H"], s["I"], s["E"], s["k"], case["T"]
        self.H, self.I, self.E, self.k = H, I, E, k
        self.x = _normal(gen, (T, H))
        # the routing that the layer's router made of its logits
        logits = torch.randn((T, E), generator=gen, device=DEV)
        if case["skew"]:
            logits = logits + 0.5 * torch.randn(E, generator=gen, device=DEV)
        p = torch.softmax(logits, dim=1)
        w, ids = torch.topk(p, k, dim=1)
        self.ids = ids.to(torch.int32)
        self.weights = (w / w.sum(dim=1, keepdim=True) if s["normalize"] else w).to(BF16)
        self.add_in = _normal(gen, (T, H), 0.5) if s["add_in"] else None
        self.codes, self.scales = _checkpoint(gen, E, 3 * I * H)
        if own:
            from pdscope_amd import layer, ops
            self.experts = ops.mxfp4_pack(self.codes, self.scales, H, I)
            self.slots = ops.slot_table([self.experts[e] for e in range(E)], DEV)
            self.ws = layer.MoEWorkspace(T, H, I, E, k, DEV)


class _Norm:
    def __init__(self, case, gen):
        T, H, k = case["T"], case["H"], case["k"]
        P = torch.float32 if case["params"] == "fp32" else BF16
        R = torch.float32 if case["resid"] == "fp32" else BF16
        if k:
            self.y = _normal(gen, (T * k, H))
            self.row_of = torch.randperm(T * k, generator=gen, device=DEV).to(torch.int32)
            self.w = torch.softmax(torch.randn((T, k), generator=gen, device=DEV), dim=1).to(BF16)
        else:
            self.block = _normal(gen, (T, H))
        self.k = k
        self.resid = _normal(gen, (T, H), 2.0, R)
        self.pre = 1 + _normal(gen, (H,), 0.1, P)
        self.post = 1 + _normal(gen, (H,), 0.1, P) if case["post"] else None
        shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[case["gate"]]
        self.gate = None if shape is None else _normal(gen, shape, 0.5, P)
        self.scale, self.eps = (0.75 if case["post"] else 1.0), 1e-6


class _Quantize:
    def __init__(self, case, gen):
        s = SHAPES[case["shape"]]
        self.H, self.I = s["H"], s["I"]
        self.experts = _weights(gen, case["E"], 3 * self.I * self.H)


STATES = {"quantize": _Quantize, "few": _Few, "grouped": _Grouped, "norm": _Norm}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(1_000_003 * (int(seed) % 1_000_000) + 17)
    return STATES[case["op"]](case, gen)


# ------------------------------------------------------------- plain forms

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _pairs(device):
    """[256, 2]: the two values of a byte of codes."""
    v = torch.tensor(_VALUES, device=device)
    return torch.stack([v.repeat(16), v.repeat_interleave(16)], dim=1)


def _dequantize(codes, scales):
    """fp32 [.., K] of codes [.., K/2] and scales [.., K/32]."""
    v = _pairs(codes.device)[codes.int()].flatten(-2).unflatten(-1, (-1, 32))
    return torch.ldexp(v, (scales.int() - 127).unsqueeze(-1)).flatten(-2)


def _quantize_plain(s):
    return _dequantize(*_quantize(s.experts)).to(BF16)


def _swiglu(x, w, I, H):
    """x [n, m, H] through the n experts w [n, 3IH] (gate | up | down), fp32."""
    g, u, d = w.split(I * H, dim=1)
    g = torch.bmm(x, g.view(-1, I, H).transpose(1, 2))
    u = torch.bmm(x, u.view(-1, I, H).transpose(1, 2))
    return torch.bmm(g / (1 + torch.exp(-g)) * u, d.view(-1, H, I).transpose(1, 2))


def _few_plain(s, lay):
    T = lay["x"].shape[0]
    logits = (lay["x"].double() @ lay["gate"].double().T).to(BF16)
    seen = logits.float() if lay["bias"] is None else logits.float() + lay["bias"]
    p = torch.exp(seen - seen.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    ids = torch.sort(seen, dim=1, descending=True, stable=True).indices[:, :s.k]
    w = p.gather(1, ids)
    w = (w / w.sum(1, keepdim=True) if s.normalize else w).to(BF16)
    at = ids.flatten()
    if s.rep == "mxfp4":
        block = _dequantize(lay["codes"][at], lay["scales"][at])
    else:
        block = lay["experts"][at].float()
    x = lay["x"].float().repeat_interleave(s.k, dim=0).unsqueeze(1)
    y = _swiglu(x, block, s.I, s.H).view(T, s.k, s.H)
    out = (y * w.float().unsqueeze(2)).sum(1)
    if lay["add_in"] is not None:
        out = out + lay["add_in"].float()
    return out.to(BF16), logits, ids.to(torch.int32), w


def _grouped_plain(s):
    """The rows of each expert, padded to the fullest one, in one batched product."""
    T = s.x.shape[0]
    flat = s.ids.flatten().long()
    counts = torch.bincount(flat, minlength=s.E)
    order = torch.argsort(flat, stable=True)
    first = torch.cumsum(counts, 0) - counts
    place = torch.arange(T * s.k, device=DEV) - first[flat[order]]
    x = torch.zeros((s.E, int(counts.max()), s.H), device=DEV)
    x[flat[order], place] = s.x[order // s.k].float()
    y = _swiglu(x, _dequantize(s.codes, s.scales), s.I, s.H)
    rows = torch.empty((T * s.k, s.H), device=DEV)
    rows[order] = y[flat[order], place]
    out = (rows.view(T, s.k, s.H) * s.weights.float().unsqueeze(2)).sum(1)
    if s.add_in is not None:
        out = out + s.add_in.float()
    return out.to(BF16)


def _norm_plain(s):
    if s.k:
        T, H = s.resid.shape
        a = (s.y[s.row_of.long()].float().view(T, s.k, H) * s.w.float().unsqueeze(2)).sum(1)
    else:
        a = s.block.float()
    if s.post is not None:
        a = a * torch.rsqrt((a * a).mean(1, keepdim=True) + s.eps) * s.post.float()
    if s.gate is not None:
        a = a * s.gate.float()
    r = s.resid.float() + s.scale * a
    n = r * torch.rsqrt((r * r).mean(1, keepdim=True) + s.eps) * s.pre.float()
    return r.to(s.resid.dtype), n.to(BF16)


# --------------------------------------------------- the framework's calls


def _run_own(s):
    from pdscope_amd import layer, ops
    if isinstance(s, _Quantize):
        blocks = ops.mxfp4_quantize(s.experts, s.H, s.I)
        return ops.mxfp4_dequantize(blocks, s.H, s.I)
    if isinstance(s, _Few):
        s.graph.replay()
        return s.outputs
    if isinstance(s, _Grouped):
        return layer.experts_resident(s.x, s.ids, s.weights, s.slots, s.ws, add_in=s.add_in, representation="mxfp4")
    if s.k:
        return ops.merge_norm_residual(s.y, s.row_of, s.w, s.resid, post_weight=s.post, gate=s.gate, scale=s.scale,
                                       pre_weight=s.pre, eps=s.eps)
    return ops.norm_residual(s.block, s.resid, post_weight=s.post, gate=s.gate, scale=s.scale, pre_weight=s.pre,
                             eps=s.eps)


def run(state):
    if own:
        return _run_own(state)
    if isinstance(state, _Quantize):
        return _quantize_plain(state)
    if isinstance(state, _Few):
        return [_few_plain(state, lay) for lay in state.layers]
    if isinstance(state, _Grouped):
        return _grouped_plain(state)
    return _norm_plain(state)


# -------------------------------------------------------------------- work


def work(case):
    """Inputs read once, outputs written once; the multiply-adds of router and
    experts.  Experts that the tokens reach: the expected number for uniform
    routing."""
    if case["op"] == "norm":
        T, H, k = case["T"], case["H"], case["k"]
        R, P = (4 if case["resid"] == "fp32" else 2), (4 if case["params"] == "fp32" else 2)
        gate = {"none": 0, "channel": H, "token": T, "full": T * H}[case["gate"]]
        byts = T * H * (2 * max(k, 1) + 2 * R + 2) + 6 * T * k + P * (H * (1 + case["post"]) + gate)
        return {"bytes": byts, "flops": T * H * (2 * k + 12)}
    s = SHAPES[case["shape"]]
    H, I, E, k = s["H"], s["I"], s["E"], s["k"]
    n = 3 * H * I
    if case["op"] == "quantize":
        return {"bytes": case["E"] * n * (4 + 2 * 17 / 32), "flops": 0}
    T = case["T"]
    touched = k if T == 1 else E * (1 - (1 - k / E) ** T)
    bits = 16 if case.get("rep") == "bf16" else 4.25
    byts = touched * n * bits / 8 + T * H * (6 if s["add_in"] else 4) + T * k * 6
    flops = 2.0 * T * k * n
    if case["op"] == "grouped":
        return {"bytes": byts, "flops": flops}
    byts += E * H * 2 + T * E * 2
    return {"bytes": byts * case["layers"], "flops": (flops + 2.0 * T * E * H) * case["layers"]}


# ------------------------------------------------------------------- exact


def _values64(codes, scales):
    """fp64 values of codes and scales, from the format: sign, two exponent
    bits (bias 1), one mantissa bit, times 2^(scale - 127)."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).long()
    e, m = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(e == 0, m * 0.5, (1 + 0.5 * m) * torch.exp2((e - 1).double()))
    v = torch.where((c & 8) != 0, -mag, mag).unflatten(-1, (-1, 32))
    return (v * torch.exp2(scales.double() - 127).unsqueeze(-1)).flatten(-2)


def _expert64(block, x, I, H):
    """x [n, H] through one expert's fp64 weights."""
    g = x @ block[:I * H].view(I, H).T
    u = x @ block[I * H:2 * I * H].view(I, H).T
    return (g * torch.sigmoid(g) * u) @ block[2 * I * H:].view(H, I).T


def _routed64(x, ids, w, I, H, block):
    """Sum over each token's experts, one expert at a time."""
    out = torch.zeros_like(x)
    for e in torch.unique(ids).tolist():
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        out.index_add_(0, t, _expert64(block(e), x[t], I, H) * w[t, slot].unsqueeze(1))
    return out


def exact(case, seed):
    """The operators in 64 bits.  The router's logits and weights are bf16 by
    definition (the layer selects by the logits and merges with the weights
    that it returns)."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "quantize":
        grid = torch.tensor(_VALUES[:8], dtype=torch.float64, device=DEV)
        # values above the midpoint of two neighbours take the upper one; at the midpoint the even code
        out = torch.empty_like(s.experts, dtype=torch.float64)
        for e in range(s.experts.shape[0]):
            b = s.experts[e].double().view(-1, 32)
            top = b.abs().amax(1, keepdim=True)
            unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -125))) - 2)
            v = (b / unit).abs()
            code = torch.zeros_like(v, dtype=torch.long)
            for i in range(7):
                mid = (grid[i] + grid[i + 1]) / 2
                code += (v > mid) | ((v == mid) & (i % 2 == 1))
            out[e] = (grid[code] * unit * torch.sign(b)).flatten()
        return out
    if case["op"] == "norm":
        r = s.resid.double()
        if s.k:
            a = torch.zeros_like(r)
            for j in range(s.k):
                a += s.w[:, j:j + 1].double() * s.y[s.row_of.view(-1, s.k)[:, j].long()].double()
        else:
            a = s.block.double()
        if s.post is not None:
            a = a / torch.sqrt(a.square().mean(1, keepdim=True) + s.eps) * s.post.double()
        r = r + s.scale * (a if s.gate is None else a * s.gate.double())
        return r, r / torch.sqrt(r.square().mean(1, keepdim=True) + s.eps) * s.pre.double()
    if case["op"] == "grouped":
        out = _routed64(s.x.double(), s.ids.long(), s.weights.double(), s.I, s.H,
                        lambda e: _values64(s.codes[e], s.scales[e]))
        return out if s.add_in is None else out + s.add_in.double()
    results = []
    for lay in s.layers:
        x = lay["x"].double()
        logits = x @ lay["gate"].double().T
        seen = logits.to(BF16).double()
        if lay["bias"] is not None:
            seen = seen + lay["bias"].double()
        p = torch.softmax(seen, dim=1)
        ids = torch.sort(seen, dim=1, descending=True, stable=True).indices[:, :s.k]
        w = p.gather(1, ids)
        if s.normalize:
            w = w / w.sum(1, keepdim=True)
        if s.rep == "mxfp4":
            out = _routed64(x, ids, w.to(BF16).double(), s.I, s.H,
                            lambda e: _values64(lay["codes"][e], lay["scales"][e]))
        else:
            out = _routed64(x, ids, w.to(BF16).double(), s.I, s.H, lambda e: lay["experts"][e].double())
        if lay["add_in"] is not None:
            out = out + lay["add_in"].double()
        results.append((out, logits, ids.to(torch.int32), w))
    return results
