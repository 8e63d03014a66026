"""CPU checks of the entry points over 8-bit rows and 4-bit matrices: sizes, limits and refusals, all of
which come before a launch (the addresses here are never read)."""
import pytest

from pdscope_amd import _lib, ops

P = 1 << 20       # an aligned address
ODD = P + 8       # one that 16 bytes do not divide


def refused(match, name, *args):
    with pytest.raises(ValueError, match=match):
        _lib.call(name, *args)


@pytest.mark.parametrize("name", ["pdscope_mxfp8_quantize", "pdscope_mxfp8_dequantize"])
def test_conversions(name):
    def call(match, x=P, codes=P, scales=P, rows=4, n=64):
        args = (x, rows, n, codes, scales) if name.endswith("_quantize") else (codes, scales, rows, n, x)
        refused(match, name, *args, None)

    for p in ("x", "codes", "scales"):
        call("null", **{p: None})
    for kw in (dict(rows=0), dict(rows=-1), dict(n=0), dict(n=33), dict(n=-32)):
        call("n % 32", **kw)
    call("too many", rows=1 << 30)
    call("16-byte", x=ODD)
    call("16-byte", codes=ODD)


def test_norms():
    def norm(match, **kw):
        a = dict(block=P, resid=P, f32=0, post=None, gate=None, rows=0, cols=0, scale=1.0, pre=None, p32=0, eps=1e-6,
                 T=4, H=256, out_resid=P, out_norm=P, codes=P, scales=P)
        a.update(kw)
        refused(match, "pdscope_norm_residual_mxfp8", *a.values(), None)

    def merged(match, **kw):
        a = dict(y=P, y_rows=8, row_of=P, w=P, k=2, add_in=None, resid=P, f32=0, post=None, gate=None, rows=0, cols=0,
                 scale=1.0, pre=None, p32=0, eps=1e-6, T=4, H=256, out_resid=P, out_norm=P, codes=P, scales=P)
        a.update(kw)
        refused(match, "pdscope_merge_norm_residual_mxfp8", *a.values(), None)

    for call, src in ((norm, "block"), (merged, "y")):
        for p in (src, "resid", "codes", "scales"):
            call("null", **{p: None})
        for kw in (dict(T=0), dict(T=1 << 22), dict(H=0), dict(H=16416)):
            call("T >= 1", **kw)
        call("H % 32", H=48)
        call("eps", eps=-1e-9)
    merged("null", row_of=None)
    merged("null", w=None)
    merged("k >= 1", k=0)
    merged("y_rows >= 1", y_rows=0)


def test_grouped():
    def call(match, **kw):
        a = dict(x=P, xs=P, perm=P, offsets=P, sel=P, nsel=4, tile_start=P, max_tiles=4, block_m=32, slots=P, H=256,
                 I=128, h=P, hs=P, y=P)
        a.update(kw)
        refused(match, "pdscope_swiglu_grouped_mxfp8", *a.values(), None)

    for p in ("x", "xs", "perm", "offsets", "sel", "tile_start", "slots", "h", "hs", "y"):
        call("null", **{p: None})
    call("nsel", nsel=0)
    for n in (0, -3, (1 << 22) + 1):
        call("max_tiles", max_tiles=n)
    for bm in (0, 16, 33, 96):
        call("block_m", block_m=bm)
    for H, I in ((192, 128), (256, 64), (0, 128), (1 << 17, 128)):
        call("H % 128", H=H, I=I)
    for p in ("x", "h", "y"):
        call("16-byte", **{p: ODD})
    for p in ("xs", "hs"):
        call("4-byte", **{p: P + 2})
    call("too many tiles", max_tiles=1 << 22, I=768)


@pytest.mark.parametrize("N,K,G,zeros", [(1, 32, 32, False), (16, 128, 128, True), (4096, 2048, 128, False), (4097, 2816, 32, True)])
def test_matrix_bytes(N, K, G, zeros):
    """Whole units of 16 rows and 128 inputs: half a byte a code, two a scale, one a zero point."""
    units = -(-N // 16) * -(-K // 128)
    assert ops.int4_bytes(N, K, G, zeros) == units * (1024 + 16 * (128 // G) * (3 if zeros else 2))


@pytest.mark.parametrize("N,K,G", [(0, 128, 32), (1 << 25, 128, 32), (16, 0, 32), (16, 144, 32), (16, 128, 16), (16, 128, 256),
                                   (16, 96, 64), (16, 1 << 21, 128), (-1, 128, 32)])
def test_no_matrix_of_other_shapes(N, K, G):
    assert _lib.load().pdscope_int4_bytes(N, K, G, 0) == 0
    with pytest.raises(ValueError, match="groups of 32"):
        ops.int4_bytes(N, K, G)
    for name, args in (("pdscope_int4_pack", (P, P, None, N, K, G, P)), ("pdscope_int4_quantize", (P, N, K, G, 0, P)),
                       ("pdscope_int4_dequantize", (P, N, K, G, 0, 0, P)),
                       ("pdscope_linear_int4", (P, P, None, 4, N, K, G, 0, 0, P))):
        refused("K % G", name, *args, None)


def test_matrices():
    refused("null", "pdscope_int4_pack", None, P, None, 16, 128, 32, P, None)
    refused("null", "pdscope_int4_pack", P, None, None, 16, 128, 32, P, None)
    refused("null", "pdscope_int4_pack", P, P, None, 16, 128, 32, None, None)
    refused("null", "pdscope_int4_quantize", None, 16, 128, 32, 0, P, None)
    refused("null", "pdscope_int4_dequantize", P, 16, 128, 32, 0, 0, None, None)
    refused("16-byte", "pdscope_int4_pack", ODD, P, None, 16, 128, 32, P, None)
    refused("16-byte", "pdscope_int4_quantize", P, 16, 128, 32, 0, ODD, None)
    refused("16-byte", "pdscope_int4_dequantize", ODD, 16, 128, 32, 0, 0, P, None)
    refused("too many weights", "pdscope_int4_quantize", P, 1 << 24, 1 << 20, 32, 0, P, None)


def test_products():
    def call(match, **kw):
        a = dict(x=P, w=P, bias=None, T=4, N=64, K=256, G=64, zeros=0, fp16=0, y=P)
        a.update(kw)
        refused(match, "pdscope_linear_int4", *a.values(), None)

    for p in ("x", "w", "y"):
        call("null", **{p: None})
    for p in ("x", "w"):
        call("16-byte", **{p: ODD})
    for T in (0, -5, (1 << 24) + 1):
        call("1 <= T", T=T)
    call("too many outputs", T=1 << 24, N=1 << 16)
