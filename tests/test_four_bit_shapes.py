"""Shapes that 4-bit experts_resident passes on to launches which trust them: refused before
the first one.  Without a GPU: tensors live on the CPU, launches are recorded."""
import pytest
import torch

from pdscope_amd import layer, ops

BF16 = torch.bfloat16
H, I, E, k, T = 256, 128, 8, 4, 20


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_need", lambda *a, **kw: None)
    monkeypatch.setattr(ops, "_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_call_on", lambda dev, name, *a: seen.append(name))
    monkeypatch.setattr(ops._lib, "call", lambda name, *a: seen.append(name))
    return seen


def call(**kw):
    def bf(*shape):
        return torch.zeros(shape, dtype=BF16)

    a = dict(x=bf(T, H), ids=(T, k), weights=(T, k), out=None, add_in=None)
    a.update(kw)
    ws = layer.MoEWorkspace(T, H, I, E, k, "cpu")
    return layer.experts_resident(a["x"], torch.zeros(a["ids"], dtype=torch.int32), bf(*a["weights"]),
                                  torch.zeros(E, dtype=torch.int64), ws,
                                  out=None if a["out"] is None else bf(*a["out"]),
                                  add_in=None if a["add_in"] is None else bf(*a["add_in"]), representation="mxfp4")


# ids of more tokens than x has, more slots than the workspace holds; weights, output and
# summand that the merge would read or write behind
@pytest.mark.parametrize("kw,match", [
    (dict(ids=(T + 1, k), weights=(T + 1, k)), "ids"), (dict(ids=(T - 1, k), weights=(T - 1, k)), "ids"),
    (dict(ids=(T, k + 1), weights=(T, k + 1)), "ids"), (dict(ids=(T * k,), weights=(T, k)), "ids"),
    (dict(ids=(T, 0), weights=(T, 0)), "ids"),
    (dict(weights=(T, k - 1)), "weights"), (dict(weights=(T + 1, k)), "weights"),
    (dict(out=(T - 1, H)), "out"), (dict(out=(T, H - 8)), "out"), (dict(out=(T * H,)), "out"),
    (dict(add_in=(T - 1, H)), "add_in"), (dict(add_in=(T, H // 2)), "add_in")])
def test_refused(launches, kw, match):
    with pytest.raises(ValueError, match=f"^{match} must be"):
        call(**kw)
    assert not launches


@pytest.mark.parametrize("kw", [{}, dict(ids=(T, k - 1), weights=(T, k - 1)), dict(out=(T, H), add_in=(T, H)),
                                dict(out=(T + 3, H), add_in=(T + 3, H))])
def test_taken(launches, kw):
    """A workspace of more slots per token, buffers of more rows."""
    call(**kw)
    assert launches == ["pdscope_pack_schedule_balanced", "pdscope_swiglu_grouped_mxfp4", "pdscope_merge"]
