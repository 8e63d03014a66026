"""CPU checks of the entry points over 4-bit experts, a few tokens and the norms:
sizes, limits and refusals, all of which come before a launch (the addresses here
are never read)."""
import pytest

from pdscope_amd import _lib, ops

P = 1 << 20       # an aligned address
ODD = P + 8       # one that 16 bytes do not divide


def refused(match, name, *args):
    with pytest.raises(ValueError, match=match):
        _lib.call(name, *args)


@pytest.mark.parametrize("H,I", [(128, 128), (2048, 768), (2048, 1408), (640, 384)])
def test_block_bytes(H, I):
    """17/32 byte a weight: a code of half a byte each, a scale byte per 32."""
    assert ops.mxfp4_block_bytes(H, I) == 3 * H * I // 2 + 3 * H * I // 32


@pytest.mark.parametrize("H,I", [(0, 128), (128, 0), (192, 128), (128, 64), (-128, 128)])
def test_no_block_of_other_shapes(H, I):
    assert _lib.load().pdscope_mxfp4_block_bytes(H, I) == 0
    with pytest.raises(ValueError, match="H % 128"):
        ops.mxfp4_block_bytes(H, I)


@pytest.mark.parametrize("name", ["pdscope_mxfp4_quantize", "pdscope_mxfp4_dequantize", "pdscope_mxfp4_pack"])
def test_conversions(name):
    two = name.endswith("pack")

    def call(match, src=P, n=1, H=128, I=128, dst=P):
        refused(match, name, *([src, src] if two else [src]), n, H, I, dst, None)

    call("null", src=None)
    call("null", dst=None)
    for n in (0, -1, 65537):
        call("1 to 65536 experts", n=n)
    for H, I in ((0, 128), (130, 128), (128, 100), (1 << 17, 128), (128, 1 << 17)):
        call("H % 128", H=H, I=I)
    call("16-byte", src=ODD)
    call("16-byte", dst=ODD)
    call("too many", n=65536, H=65536, I=65536)


def test_grouped():
    def call(match, **kw):
        a = dict(x=P, perm=P, offsets=P, sel=P, nsel=4, tile_start=P, max_tiles=4, block_m=32, slots=P, H=256, I=128,
                 h=P, y=P)
        a.update(kw)
        refused(match, "pdscope_swiglu_grouped_mxfp4", *a.values(), None)

    for p in ("x", "perm", "offsets", "sel", "tile_start", "slots", "h", "y"):
        call("null", **{p: None})
    call("nsel", nsel=0)
    for n in (0, -3, (1 << 22) + 1):
        call("max_tiles", max_tiles=n)
    for bm in (0, 16, 33, 128):
        call("block_m", block_m=bm)
    for H, I in ((192, 128), (256, 64), (0, 128), (1 << 17, 128)):
        call("H % 128", H=H, I=I)
    for p in ("x", "h", "y"):
        call("16-byte", **{p: ODD})
    call("too many tiles", max_tiles=1 << 22, I=768)
    assert [ops.grouped_mxfp4_block_m(r) for r in (0, 1, 16, 17, 256)] == [32, 32, 32, 64, 64]


def test_a_few_tokens():
    for T, H, I, E, k, ok in ((1, 2048, 768, 128, 8, 1), (16, 4096, 128, 256, 16, 1), (17, 2048, 768, 128, 8, 0),
                              (0, 128, 128, 4, 1, 0), (1, 4224, 128, 4, 1, 0), (1, 192, 128, 4, 1, 0),
                              (1, 128, 96, 4, 1, 0), (1, 128, 128, 257, 1, 0), (1, 128, 128, 4, 5, 0),
                              (1, 128, 128, 64, 17, 0), (1, 128, 128, 4, 0, 0)):
        assert ops.moe_few_supported(T, H, I, E, k) is bool(ok)
        size = ops.moe_few_workspace_size(T, H, I, E, k)
        # a partial row of fp32 for every token, slot and chunk of 32 columns
        assert size >= T * k * (I // 32) * H * 4 if ok else size == 0

    def call(match, **kw):
        a = dict(x=P, gate=P, bias=None, T=4, H=256, E=8, k=2, normalize=1, slots=P, mxfp4=1, I=128, add_in=None,
                 logits=P, ids=P, weights=P, out=P, workspace=P)
        a.update(kw)
        refused(match, "pdscope_moe_few", *a.values(), None)

    for p in ("x", "gate", "slots", "logits", "ids", "weights", "out", "workspace"):
        call("null", **{p: None})
    for p in ("x", "gate", "workspace"):
        call("16-byte", **{p: ODD})
    for kw in (dict(T=0), dict(T=17), dict(H=130), dict(H=4224), dict(I=64), dict(E=0), dict(E=257), dict(k=0),
               dict(k=9), dict(E=64, k=17)):
        call("need 1 <= T <= 16", **kw)


def test_norms():
    def norm(match, **kw):
        a = dict(block=P, resid=P, f32=0, post=None, gate=None, rows=0, cols=0, scale=1.0, pre=None, p32=0, eps=1e-6,
                 T=4, H=256, out_resid=P, out_norm=P)
        a.update(kw)
        refused(match, "pdscope_norm_residual", *a.values(), None)

    def merged(match, **kw):
        a = dict(y=P, y_rows=8, row_of=P, w=P, k=2, add_in=None, resid=P, f32=0, post=None, gate=None, rows=0, cols=0,
                 scale=1.0, pre=None, p32=0, eps=1e-6, T=4, H=256, out_resid=P, out_norm=P)
        a.update(kw)
        refused(match, "pdscope_merge_norm_residual", *a.values(), None)

    for call, src in ((norm, "block"), (merged, "y")):
        call("null", **{src: None})
        call("null", resid=None)
        call("null", out_resid=None, out_norm=None)
        for kw in (dict(T=0), dict(T=-1), dict(T=1 << 22), dict(H=0), dict(H=16385)):
            call("T >= 1", **kw)
        call("eps", eps=-1e-9)
        call("eps", eps=float("nan"))
    merged("null", row_of=None)
    merged("null", w=None)
    merged("k >= 1", k=0)
    merged("y_rows >= 1", y_rows=0)
