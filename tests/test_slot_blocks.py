"""A slot table remembers the blocks that slot_table made it of, and every entry point that
takes one refuses it for experts of another representation or shape, whose blocks its kernels
would read past the end of.  On the CPU: nothing here gets as far as a launch."""
import pytest
import torch

from pdscope_amd import layer, ops

BF16 = torch.bfloat16
H, I, E, k, T = 256, 128, 4, 2, 3
FOUR, TWO = ops.mxfp4_block_bytes(H, I), 6 * H * I  # bytes of a 4-bit and a bf16 expert


def table(rep, n=E, H=H, I=I):
    if rep == "mxfp4":
        blocks = torch.zeros((n, ops.mxfp4_block_bytes(H, I)), dtype=torch.uint8)
    else:
        blocks = torch.zeros((n, 3 * I * H), dtype=BF16)
    return ops.slot_table([blocks[e] for e in range(n)], "cpu")


@pytest.fixture
def host(monkeypatch):
    """The entry points without a GPU: tensors may live on the CPU, and a launch is an error."""
    def launched(*a):
        raise AssertionError(f"launched {a}")

    monkeypatch.setattr(ops, "_need", lambda *a, **kw: None)
    monkeypatch.setattr(ops, "pack", lambda *a, **kw: None)
    monkeypatch.setattr(ops, "route_topk", lambda *a, **kw: None)
    monkeypatch.setattr(ops, "decode_layer_supported", lambda *a: False)
    monkeypatch.setattr(ops, "_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_call_on", launched)
    monkeypatch.setattr(ops._lib, "call", launched)


class Args:
    def __init__(self):
        self.ws = layer.MoEWorkspace(T, H, I, E, k, "cpu", few_tokens=True)
        self.x = torch.zeros((T, H), dtype=BF16)
        self.gate = torch.zeros((E, H), dtype=BF16)
        self.ids = torch.zeros((T, k), dtype=torch.int32)
        self.w = torch.zeros((T, k), dtype=BF16)


def calls(a, slots, rep):
    """Every call of this representation that takes a slot table, for one token and several."""
    ws, x, one = a.ws, a.x, a.x[:1]
    out = [lambda: layer.moe_few(x, a.gate, slots, ws, representation=rep),
           lambda: layer.moe_few(one, a.gate, slots, ws, representation=rep),
           lambda: layer.moe_forward(x, a.gate, slots, ws, representation=rep),
           lambda: layer.moe_forward(one, a.gate, slots, ws, representation=rep),
           lambda: layer.moe_forward(x, a.gate, slots, ws, merge="reference", representation=rep),
           lambda: layer.experts_resident(x, a.ids, a.w, slots, ws, representation=rep),
           lambda: layer.experts_resident(one, a.ids[:1], a.w[:1], slots, ws, representation=rep)]
    grouped = (ws.sel_all, ws.tile_start, 4, 32)
    if rep == "mxfp4":
        return out + [lambda: ops.swiglu_grouped_mxfp4(x, ws.perm_token, ws.offsets, *grouped, slots, H, I, ws.h_ws, ws.y)]
    logits, ids, w, _ = ws.views(1)
    one_token = dict(out=ws.out[:1], logits=logits, ids=ids, weights=w, h_ws=ws.h_ws)
    return out + [
        lambda: layer.shared_forward(x, slots, layer.MoEWorkspace(T, H, I, E, k, "cpu", shared_I=I)),
        lambda: ops.swiglu_grouped(x, ws.perm_token, ws.offsets, *grouped, slots, H, I, ws.h_ws, ws.y),
        lambda: ops.swiglu_grouped_gateup(x, ws.perm_token, ws.offsets, *grouped, slots, H, I, ws.h_ws),
        lambda: ops.swiglu_grouped_down(ws.h_ws, ws.offsets, *grouped, slots, H, I, ws.y),
        lambda: ops.swiglu_grouped_layer(x, ws.perm_token, ws.offsets, *grouped, ws.tile_start, 4, 32, slots, H, I,
                                         ws.h_ws, ws.y),
        lambda: ops.swiglu_decode(one, a.ids[:1], a.w[:1], slots, H, I, ws.h_ws, ws.out[:1]),
        lambda: ops.decode_shared_layer(one, a.gate, slots, I, k, True, slots, I, h_shared=ws.h_ws,
                                        y_shared=ws.y[:H].view(1, H), workspace=ws.route_ws, **one_token),
        lambda: ops.decode_layer(one, a.gate, slots, I, k, True, **one_token),
        lambda: ops.DecodeBinding(a.gate, slots, I, k, True, host=torch.zeros(8, dtype=torch.int32), error_at=7)]


@pytest.mark.parametrize("i", range(16))
def test_four_bit_blocks_are_not_read_as_bf16(host, i):
    """Also through a view of the table, and where the representation is left to its default."""
    a, slots = Args(), table("mxfp4", E + 1)
    for s in (slots, slots[:E]):
        every = calls(a, s, "bf16")
        assert len(every) == 16
        with pytest.raises(ValueError, match=f"blocks of {FOUR} bytes, bf16 experts .* have {TWO}"):
            every[i]()
    with pytest.raises(ValueError, match="slots address blocks"):
        layer.moe_few(a.x, a.gate, slots, a.ws)


@pytest.mark.parametrize("i", range(8))
def test_bf16_blocks_are_not_read_as_four_bit(host, i):
    every = calls(Args(), table("bf16"), "mxfp4")
    assert len(every) == 8
    with pytest.raises(ValueError, match="blocks of torch.bfloat16"):
        every[i]()


@pytest.mark.parametrize("rep", ["bf16", "mxfp4"])
def test_blocks_of_a_smaller_shape(host, rep):
    for call in calls(Args(), table(rep, I=I // 2 if rep == "bf16" else 128, H=H if rep == "bf16" else 128), rep):
        with pytest.raises(ValueError, match="slots address blocks"):
            call()


def test_a_shared_block_of_a_smaller_shape(host):
    a = Args()
    ws = layer.MoEWorkspace(T, H, I, E, k, "cpu", shared_I=2 * I)
    with pytest.raises(ValueError, match="slots address blocks"):
        layer.moe_forward(a.x, a.gate, table("bf16"), ws, shared_slot=table("bf16", 1))


def test_tables_that_pass():
    """Blocks of the right kind, with missing ones among them and larger ones beside them, a
    mixed table for neither, and tables whose blocks nobody recorded."""
    for rep in ("bf16", "mxfp4"):
        ops.check_slots(table(rep), H, I, rep)
    some = torch.zeros((2, 3 * I * H), dtype=BF16)
    ops.check_slots(ops.slot_table([some[0], some[:0], some[1]], "cpu"), H, I)
    ops.check_slots(ops.slot_table([some, some[1]], "cpu"), H, I)
    ops.check_slots(ops.slot_table([some[0].view(torch.uint8)], "cpu"), H, I)  # bf16 experts kept as bytes
    gate = [some[e, :I * H].view(I, H) for e in range(2)]  # the first matrix of each block
    ops.check_slots(ops.slot_table(gate, "cpu"), H, I)
    with pytest.raises(ValueError, match="slots address blocks"):
        ops.check_slots(ops.slot_table([some[1, 8:]], "cpu"), H, I)
    mixed = ops.slot_table([some[0], torch.zeros(FOUR, dtype=torch.uint8)], "cpu")
    for rep in ("bf16", "mxfp4"):
        with pytest.raises(ValueError, match="slots address blocks"):
            ops.check_slots(mixed, H, I, rep)
    for free in (torch.zeros(E, dtype=torch.int64), table("mxfp4").clone(), ops.slot_table([], "cpu")):
        ops.check_slots(free, H, I)
    empty = ops.slot_table([some[:0]], "cpu")
    assert empty.tolist() == [0]
