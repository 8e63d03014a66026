"""The documented run on 8-bit rows and 4-bit matrices, from a projection before a layer to the
vocabulary head behind it, eager, on another stream and captured; and measured requests of a
model on 4-bit matrices."""
import json

import pytest
import torch

from moe64 import assert_within
from pdscope_amd import layer, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
U, B = 2.0 ** -24, 2.0 ** -8


class Step:
    """One block of a serving step: projection, norm, layer, merge with the next norm, head."""

    def __init__(self, T, seed):
        self.H, self.I, self.E, self.k, self.T = 512, 256, 32, 4, T
        H, I, E, k = self.H, self.I, self.E, self.k
        g = torch.Generator(device=DEV).manual_seed(seed)
        n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
        self.attended, self.resid = n(T, 384).to(BF16), n(T, H)
        self.o_proj = ops.int4_quantize((0.05 * n(H, 384)).to(BF16), 64, True)
        self.head = ops.int4_quantize((0.05 * n(1003, H)).to(BF16), 128)
        self.gate, self.w1, self.w2 = (0.05 * n(E, H)).to(BF16), (1 + 0.1 * n(H)).to(BF16), (1 + 0.1 * n(H)).to(BF16)
        self.blocks = ops.mxfp4_quantize((0.05 * n(E, 3 * I * H)).to(BF16), H, I)
        self.slots = ops.slot_table([self.blocks[e] for e in range(E)], DEV)
        self.ws = layer.MoEWorkspace(T, H, I, E, k, DEV, mxfp8=True)

    def run(self):
        block = ops.linear_int4(self.attended, self.o_proj)
        resid, x, rows = ops.norm_residual(block, self.resid, pre_weight=self.w1, want_mxfp8=True)
        out, _, _, weights = layer.moe_forward(x, self.gate, self.slots, self.ws, representation="mxfp4",
                                               activations="mxfp8", x_rows=rows)
        resid, x, rows = ops.merge_norm_residual(self.ws.y, self.ws.views(self.T)[3].row_of, weights, resid,
                                                 pre_weight=self.w2, want_mxfp8=True)
        return out, resid, x, rows.codes.view(torch.uint8), rows.scales, ops.linear_int4(x, self.head)


@pytest.mark.parametrize("T", [1, 9, 40, 700])
def test_the_documented_run(T):
    s = Step(T, seed=T)
    want = [t.clone() for t in s.run()]
    # the head against 64 bits on its input; the layer's and the norms' outputs have tests of their own
    x, values = want[2].double(), ops.int4_dequantize(s.head).double()
    mass = x.abs() @ (values.abs() + 16 * values.abs().unflatten(1, (-1, 128)).amax(2).repeat_interleave(128, 1)).T
    assert_within(want[5], x @ values.T, B * (x.abs() @ values.abs().T) + (128 + 2 * 4 + 24) * U * mass + B * (x @ values.T).abs())
    # rows quantised in the call are those of the bf16 norm, not of the unrounded one: a code apart at most
    out2 = layer.moe_forward(want[2], s.gate, s.slots, s.ws, representation="mxfp4", activations="mxfp8")[0]
    assert out2.shape == (T, s.H) and torch.isfinite(out2.float()).all()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.run()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.run()
    for _ in range(3):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_steps_on_two_streams():
    """Two steps with workspaces of their own that may run together."""
    steps = [Step(33, seed=3), Step(120, seed=4)]
    want = [[t.clone() for t in s.run()] for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    for q in streams:
        q.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = []
        for q, s in zip(streams, steps):
            with torch.cuda.stream(q):
                got.append(s.run())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for p, q in zip(a, b):
                assert torch.equal(p, q)


def test_measured_requests_on_four_bit_matrices(tmp_path):
    """pdscope_amd.compare with int4_group: requests complete, and the same prompt gives the same tokens."""
    from pdscope_amd import compare
    model = compare.random_qwen3_moe(2, vocab_size=512, hidden_size=256, intermediate_size=512,
                                     moe_intermediate_size=128, num_attention_heads=4, num_key_value_heads=2,
                                     head_dim=64, num_experts=32, num_experts_per_tok=4)
    with torch.no_grad():
        for d in model.model.layers:
            d.mlp.gate.weight.normal_(0.0, 0.5)
    specs = compare.build_cases([24], repetitions=1, output_tokens=3, warmups=1, demand_slots=4, merge="fused")
    out = tmp_path / "run" / "result.json"
    result = compare.run(model, specs, output=out, argv=["test"], config=dict(test=True), model_name="tiny",
                         hot_per_layer=8, speculative_slots=4, demand_slots=4, merge="fused", int4_group=64)
    assert json.loads(out.read_text())["status"] == "completed"
    assert len(result["requests"]) >= 1
    reqs = [json.loads(x) for x in (out.parent / "requests.jsonl").read_text().splitlines()]
    assert len(reqs) == 2 and len({tuple(r["generated_ids"]) for r in reqs}) == 1
