"""Calls whose tensors live on another device than the current one: the launch is made with theirs current,
on its stream.  One device is enough: the current one is said to be another."""
import pytest
import torch

from pdscope_amd import layer, ops
from test_gpu_grouped_mxfp8 import make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def test_every_call_of_a_step_on_four_bits(monkeypatch):
    T, H, I, E, k = 40, 256, 128, 8, 2
    rows, ids, w, blocks, slots = make(T, H, I, E, k, seed=5)
    g = torch.Generator(device=DEV).manual_seed(6)
    n = lambda *s: torch.randn(s, generator=g, device=DEV).to(BF16)  # noqa: E731
    matrix, x, block, resid = 0.05 * n(96, H), n(T, H), n(T, H), n(T, H)
    spaces = [layer.MoEWorkspace(T, H, I, E, k, DEV, y_dtype=t) for t in (BF16, torch.float32)]

    def step():
        out = []
        for ws in spaces:
            y = layer.experts_resident(rows, ids, w, slots, ws, out=torch.empty_like(x), representation="mxfp4")
            out += [y, *ops.merge_norm_residual(ws.y, ws.views(T)[3].row_of, w, resid)]
        q = ops.int4_quantize(matrix, 64, True)
        packed = ops.pack(ids, E)
        r, m, mx = ops.norm_residual(block, resid, want_mxfp8=True)
        back = ops.mxfp8_dequantize(ops.mxfp8_quantize(x))
        return out + [q.units, ops.int4_dequantize(q), ops.linear_int4(x, q), packed.row_of, packed.offsets, r, m,
                      mx.codes.view(torch.uint8), mx.scales, back]

    want = [t.clone() for t in step()]
    entered, real = [], torch.cuda.device
    monkeypatch.setattr(ops, "_current_device", lambda: torch.cuda.current_device() + 1)

    class Device(real):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

    monkeypatch.setattr(torch.cuda, "device", Device)
    got = step()
    # pack, the grouped launches, merge and the merge with the norm twice; quantise, pack, norm, there and back, dequantise, product
    assert entered == [x.device.index] * (4 * 2 + 7)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
