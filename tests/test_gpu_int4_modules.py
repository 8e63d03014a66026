"""Linear modules on 4-bit weights in the place of a model's own: what is refused before a
module is replaced, and the inputs that a plain linear module takes."""
import pytest
import torch

from pdscope_amd import ops
from pdscope_amd.hf import Int4Linear, install_int4_linears

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def linear(k, n, bias=False, seed=1):
    torch.manual_seed(seed)
    return torch.nn.Linear(k, n, bias=bias).to(BF16).to(DEV)


def test_a_bias_of_another_type_or_device_is_refused_before_anything_is_replaced():
    for change in (lambda b: b.float(), lambda b: b.cpu(), lambda b: b.half()):
        model = torch.nn.Sequential(linear(128, 64, True), linear(64, 32, True))
        model[1].bias = torch.nn.Parameter(change(model[1].bias.detach()))
        before = list(model)
        with pytest.raises(ValueError, match="bias"):
            install_int4_linears(model, 64)
        assert all(a is b for a, b in zip(model, before))


def test_contiguous_inputs_at_addresses_that_16_bytes_do_not_divide():
    q = Int4Linear.of(linear(128, 48, True), 64)
    for shape in ((3, 128), (2, 40, 128)):
        n = torch.Size(shape).numel()
        x = torch.randn(n, device=DEV).to(BF16)
        want = q(x.view(shape))
        for off in (1, 2, 4):
            room = torch.empty(n + off, dtype=BF16, device=DEV)
            room[off:] = x
            at = room[off:].view(shape)
            assert at.is_contiguous() and at.data_ptr() % 16
            assert torch.equal(q(at), want)


def test_autocast():
    """Where autocast makes bf16 of a linear module's inputs, so it does of this one's; elsewhere
    inputs of other types are refused as they are without it."""
    q = Int4Linear.of(linear(128, 48, True), 64)
    x = torch.randn((5, 128), device=DEV)
    want = q(x.to(BF16))
    with torch.autocast("cuda", dtype=BF16):
        for t in (x, x.to(BF16), x.to(BF16).float()):
            y = q(t)
            assert y.dtype is BF16 and torch.equal(y, want)
        y = q(x.half())
        assert y.dtype is BF16 and torch.equal(y, q(x.half().to(BF16)))
        with pytest.raises(ValueError, match="bfloat16"):
            q(x.double())  # a plain module leaves 64 bits as they are too, and refuses the mixture
        with torch.autocast("cuda", enabled=False), pytest.raises(ValueError, match="bfloat16"):
            q(x)
        with pytest.raises(RuntimeError, match="no gradient"):
            q(x.clone().requires_grad_())
    with torch.autocast("cuda", dtype=torch.float16), pytest.raises(ValueError, match="bfloat16"):
        q(x)
    with pytest.raises(ValueError, match="bfloat16"):
        q(x)


class Shared(torch.nn.Module):
    def __init__(self, shared):
        super().__init__()
        self.first, self.inner = shared, torch.nn.Sequential(linear(64, 64, seed=2), shared)
        self.mlp = torch.nn.Module()
        self.mlp.gate, self.mlp.up = linear(64, 32, seed=3), linear(64, 32, seed=4)
        self.up_again = self.mlp.up


def test_a_module_under_two_names():
    """Both names get the one 4-bit form; a module that one name keeps, or that an expert block has
    too, stays under all of its names."""
    model = Shared(linear(64, 64))
    up, gate = model.mlp.up, model.mlp.gate
    assert sorted(install_int4_linears(model, 64)) == ["first", "inner.0", "inner.1"]
    assert type(model.first) is Int4Linear and model.first is model.inner[1] and model.inner[0] is not model.first
    assert model.mlp.up is up and model.up_again is up and model.mlp.gate is gate
    model = Shared(linear(64, 64))
    first = model.first
    assert install_int4_linears(model, 64, keep=("inner.1",)) == ["inner.0"]
    assert model.first is first and model.inner[1] is first
