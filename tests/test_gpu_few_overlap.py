"""The buffers that the layer of a few tokens may share with its output: the summand alone, the
activations alone; both are tested beside the layer itself."""
import pytest
import torch

from pdscope_amd import layer
from test_gpu_few import Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared", ["add_in", "x"])
@pytest.mark.parametrize("rep", ["mxfp4", "bf16"])
@pytest.mark.parametrize("T,H", [(1, 512), (7, 640), (16, 2048)])
def test_a_buffer_that_the_output_takes(T, H, rep, shared):
    lay = Layer(T, H, 256, 16, 4, rep, add_in=True, seed=T)
    want = [t.clone() for t in lay.run()]
    for _ in range(3):
        buf = lay.ws.out[:T]
        buf.copy_(getattr(lay, shared))
        args = dict(x=lay.x, add_in=lay.add_in)
        args[shared] = buf
        got = layer.moe_few(args["x"], lay.gate, lay.slots, lay.ws, add_in=args["add_in"], representation=rep)
        assert got[0].data_ptr() == buf.data_ptr()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
