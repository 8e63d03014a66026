"""Slot tables longer and shorter than the experts of a 4-bit prompt, without a GPU: tensors
live on the CPU, and what would be launched is recorded instead."""
import pytest
import torch

from pdscope_amd import layer, ops

BF16 = torch.bfloat16
H, I, E, k, T = 256, 128, 4, 2, 20


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_need", lambda *a, **kw: None)
    monkeypatch.setattr(ops, "_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_call_on", lambda dev, name, *a: seen.append(name))
    monkeypatch.setattr(ops._lib, "call", lambda name, *a: seen.append(name))
    return seen


def run(entries, offsets=E + 1):
    """experts_resident and the grouped call alone over a table of `entries`."""
    ws = layer.MoEWorkspace(T, H, I, E, k, "cpu")
    slots = torch.zeros(entries, dtype=torch.int64)
    x, ids = torch.zeros((T, H), dtype=BF16), torch.zeros((T, k), dtype=torch.int32)
    w = torch.zeros((T, k), dtype=BF16)
    return (lambda: layer.experts_resident(x, ids, w, slots, ws, representation="mxfp4"),
            lambda: ops.swiglu_grouped_mxfp4(x, ws.perm_token, torch.zeros(offsets, dtype=torch.int32), ws.sel_all,
                                             ws.tile_start, 4, 32, slots, H, I, ws.h_ws, ws.y))


@pytest.mark.parametrize("entries", [E, E + 1, 3 * E])
def test_a_table_with_an_entry_per_expert(launches, entries):
    """Further entries are not read: moe_few takes such a table too."""
    for call in run(entries):
        launches.clear()
        call()
        assert "pdscope_swiglu_grouped_mxfp4" in launches


@pytest.mark.parametrize("entries", [0, 1, E - 1])
def test_a_shorter_table(launches, entries):
    """The schedule's experts go up to E - 1: the kernel would read addresses behind the table."""
    for call in run(entries):
        with pytest.raises(ValueError, match="one entry per expert"):
            call()
    assert "pdscope_swiglu_grouped_mxfp4" not in launches


def test_offsets_without_an_end(launches):
    with pytest.raises(ValueError, match="offsets"):
        run(E, offsets=0)[1]()
