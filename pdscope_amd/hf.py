"""A transformers Qwen3-MoE model driven through PDScopeCudaRuntime (the model
hook-up of benchmarks/pdscope_compare.py:181-212 and forward_layer :285-304).

``install_expert_blocks(model, forward_layer)`` replaces every decoder
layer's sparse MoE block by an ``ExpertBlock`` that keeps only the router
weight and calls ``forward_layer(layer, hidden, gate_weight)``.  The block
returns ``(out, router_logits)`` where the installed transformers decoder
unpacks a pair (4.x) and ``out`` where it takes a tensor (5.x).

``ModelSession(model, ...)`` is that driver: it takes the model's expert
masters (``collect_model_experts``), packs them into pooled pinned blocks,
installs the blocks, moves the rest of the model to the GPU and creates the
runtime with a static hot set; ``forward_layer`` feeds each layer call with
the caller's step (``session.step``: 0 for the prompt, then 1, 2, ... per
decoded token) and the next layer's router for the gate-fallback prefetch,
and keeps the runtime's per-layer trace rows.

``install_int4_linears(model)`` replaces the linear modules that stay outside the
expert blocks (the attention's projections, the vocabulary head) by ``Int4Linear``:
4-bit codes with a scale per group of inputs, a little over a quarter of the bytes
that a decoded token reads of them in bf16 (the reference keeps them as they are).
``ModelSession(model, int4_group=128, ...)`` does so at start.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import ops
from .cache import ExpertKey
from .checkpoint import collect_model_experts, pin_cpu_master_storage
from .pdscope_runtime import PDScopeCudaRuntime


class ExpertBlock(torch.nn.Module):
    """Stand-in for a decoder layer's sparse MoE block (pdscope_compare.py:198-200)."""

    def __init__(self, gate, layer, forward_layer, return_router_logits):
        super().__init__()
        self.gate, self.layer = gate, layer
        self._forward_layer = forward_layer
        self.return_router_logits = return_router_logits

    def forward(self, hidden):
        out, logits = self._forward_layer(self.layer, hidden, self.gate.weight)
        return (out, logits) if self.return_router_logits else out


def _returns_pair():
    import transformers
    return int(transformers.__version__.split(".")[0]) < 5


def install_expert_blocks(model, forward_layer, *, return_router_logits=None):
    """Replace every sparse MoE block; returns {layer: original block}."""
    if return_router_logits is None:
        return_router_logits = _returns_pair()
    originals = {}
    for layer, decoder in enumerate(model.model.layers):
        if not hasattr(decoder.mlp, "experts") or not hasattr(decoder.mlp, "gate"):
            raise ValueError("dense layers require a separate adapter")
        originals[layer] = decoder.mlp
        decoder.mlp = ExpertBlock(decoder.mlp.gate, layer, forward_layer, return_router_logits)
    return originals


class Int4Linear(torch.nn.Module):
    """A linear module over a 4-bit matrix (ops.Int4Weight): bf16 inputs [..., K] on the
    matrix' device (under autocast to bf16 fp32 and fp16 ones too) to bf16 outputs
    [..., N].  Inference only: ops.linear_int4 has no gradient, of reverse or forward
    mode."""

    def __init__(self, weight: ops.Int4Weight, bias=None):
        super().__init__()
        self.register_buffer("units", weight.units)
        self.register_buffer("bias", bias)
        self.in_features, self.out_features = weight.K, weight.N
        self._shape = (weight.N, weight.K, weight.group, weight.zeros, weight.scale_dtype)

    @classmethod
    def of(cls, linear: torch.nn.Linear, group=128, zeros=False):
        """The 4-bit form of a bf16 linear module on the GPU (ops.int4_quantize)."""
        bias = None if linear.bias is None else linear.bias.detach()
        return cls(ops.int4_quantize(linear.weight.detach().contiguous(), group, zeros), bias)

    @property
    def weight4(self) -> ops.Int4Weight:
        return ops.Int4Weight(self.units, *self._shape)

    def forward(self, x):
        if torch.is_grad_enabled() and x.requires_grad or forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError("Int4Linear has no gradient: run it under torch.no_grad() or inference_mode()")
        # under autocast to bf16 the inputs that it casts for a plain linear module
        if x.dtype in (torch.float32, torch.float16) and x.is_cuda and torch.is_autocast_enabled("cuda") \
                and torch.get_autocast_dtype("cuda") is torch.bfloat16:
            x = x.to(torch.bfloat16)
        rows = x.reshape(-1, x.shape[-1]).contiguous()
        if rows.data_ptr() % 16:  # the kernels read 16 bytes at a time
            rows = rows.clone()
        out = ops.linear_int4(rows, self.weight4, bias=self.bias)
        return out.view(*x.shape[:-1], self.out_features)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, group={self._shape[2]}"


def install_int4_linears(model, group=128, zeros=False, keep=()):
    """Replace every torch.nn.Linear of a model that is on the GPU, but for routers and
    experts (modules below a `mlp` with a `gate`) and the names in `keep`, by its
    4-bit form; returns the replaced modules' names.  A module that the model has under
    several names gets one 4-bit form for all of them, or stays under all where one is
    an expert block's or in `keep`.  Their bf16 weights are freed
    where nothing else holds them (a tied embedding does)."""
    if group not in (32, 64, 128):
        raise ValueError(f"group must be 32, 64 or 128, got {group}")
    if type(model) is torch.nn.Linear:
        raise ValueError("the model is a linear module itself, which no parent holds: take Int4Linear.of")
    named = list(model.named_modules(remove_duplicate=False))
    kept = {id(m) for n, m in named if n in keep}
    for n, m in named:
        if hasattr(m, "gate") and n.rsplit(".", 1)[-1] == "mlp":
            kept.update(id(part) for part in m.modules())
    found = [(n, m) for n, m in named if type(m) is torch.nn.Linear and id(m) not in kept]
    for name, m in found:  # before anything is replaced
        if m.weight.dtype != torch.bfloat16 or m.weight.device.type != "cuda":
            raise ValueError(f"{name} must be bf16 on the GPU, got {m.weight.dtype} on {m.weight.device}")
        if m.bias is not None and (m.bias.dtype != m.weight.dtype or m.bias.device != m.weight.device):
            raise ValueError(f"{name}'s bias must be as its weight, bf16 on {m.weight.device}, got {m.bias.dtype} on "
                             f"{m.bias.device}")
        if m.in_features % group:
            raise ValueError(f"{name} has {m.in_features} inputs, not whole groups of {group}: keep it or take smaller groups")
    forms = {}
    for name, m in found:
        if id(m) not in forms:
            forms[id(m)] = Int4Linear.of(m, group, zeros)
        parent, _, leaf = name.rpartition(".")
        setattr(model.get_submodule(parent) if parent else model, leaf, forms[id(m)])
    return [n for n, _ in found]


class ModelSession:
    """Qwen3-MoE model whose expert layers run on the gfx950 path.

    hot_per_layer: experts per layer placed in the static hot set (the first
    ones of ``hot_order[layer]`` when given, else ids 0, 1, ...);
    speculative_slots, demand_slots and the other keywords go to
    PDScopeCudaRuntime.  int4_group (32, 64 or 128): the linear modules outside the
    expert blocks run on 4-bit weights (install_int4_linears)."""

    def __init__(self, model, *, hot_per_layer, speculative_slots, demand_slots=2, hot_order=None,
                 device=0, block_cap_bytes=256 * 1024**2, int4_group=None, **runtime_kwargs):
        if model.config.model_type != "qwen3_moe":
            raise ValueError("only Qwen3 MoE supported")
        self.model = model
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        self.top_k = model.config.num_experts_per_tok
        self.normalize = bool(model.config.norm_topk_prob)
        self.masters = collect_model_experts(model)
        self.pinned = pin_cpu_master_storage(self.masters, block_cap_bytes=block_cap_bytes)
        self.gates = {}
        install_expert_blocks(model, self.forward_layer)
        for layer, decoder in enumerate(model.model.layers):
            self.gates[layer] = decoder.mlp.gate
        model.to(self.device)
        self.int4_linears = [] if int4_group is None else install_int4_linears(model, int4_group)
        E = model.config.num_experts
        hot = []
        for layer in self.gates:
            order = list(hot_order[layer]) if hot_order is not None else list(range(E))
            hot += [ExpertKey(layer, e, "bf16") for e in order[:hot_per_layer]]
        self.runtime = PDScopeCudaRuntime(self.masters, hot_keys=hot, speculative_slots=speculative_slots,
                                          device=self.device.index, demand_slots=demand_slots, **runtime_kwargs)
        self.step = 0
        self.request = "pdscope"
        self.traces = []

    def forward_layer(self, layer, hidden, gate):
        shape = hidden.shape
        x = hidden.reshape(-1, shape[-1])
        nxt = self.gates.get(layer + 1)
        out, routing, row = self.runtime.forward(x, gate, layer=layer, step=self.step, request=self.request,
                                                 next_gate=None if nxt is None else nxt.weight,
                                                 top_k=self.top_k, normalize=self.normalize)
        if sum(row["token_counts"].values()) != x.shape[0] * self.top_k:
            raise AssertionError("missing routed assignment")
        self.traces.append(row)
        return out.reshape(shape), routing.logits

    def close(self):
        self.runtime.close()
