"""CPU checks of the entry points over fp32 rows: refusals that come before a launch (the addresses here
are never read)."""
import pytest

from pdscope_amd import _lib

P = 1 << 20       # an aligned address
ODD = P + 8       # one that 16 bytes do not divide


def refused(match, name, a, **kw):
    with pytest.raises(ValueError, match=match):
        _lib.call(name, *{**a, **kw}.values(), None)


def test_merge():
    a = dict(y=P, row_of=P, w=P, T=4, k=2, H=64, add_in=None, out=P)
    for p in ("y", "row_of", "w", "out"):
        refused("null", "pdscope_merge_y32", a, **{p: None})
    for kw in (dict(T=0), dict(k=0), dict(H=0), dict(H=12), dict(H=-8)):
        refused("H % 8", "pdscope_merge_y32", a, **kw)


def test_merge_and_norm():
    a = dict(y=P, y_rows=8, row_of=P, w=P, k=2, add_in=None, resid=P, f32=0, post=None, gate=None, rows=0, cols=0, scale=1.0,
             pre=None, p32=0, eps=1e-6, T=4, H=256, out_resid=P, out_norm=P, codes=P, scales=P)
    name = "pdscope_merge_norm_residual_y32"
    for kw in (dict(y=None), dict(row_of=None), dict(w=None), dict(resid=None), dict(codes=None), dict(scales=None),
               dict(out_resid=None, out_norm=None, codes=None, scales=None)):
        refused("null", name, a, **kw)
    for kw in (dict(T=0), dict(T=1 << 22), dict(H=0), dict(H=16416)):
        refused("T >= 1", name, a, **kw)
    refused("H % 32", name, a, H=48)
    refused("eps", name, a, eps=-1e-9)
    refused("k >= 1", name, a, k=0)
    refused("y_rows >= 1", name, a, y_rows=0)


def test_grouped():
    a = dict(x=P, xs=P, perm=P, offsets=P, sel=P, nsel=4, tile_start=P, max_tiles=4, block_m=32, slots=P, H=256, I=128, h=P,
             hs=P, y=P)
    name = "pdscope_swiglu_grouped_mxfp8_y32"
    for p in ("x", "xs", "perm", "offsets", "sel", "tile_start", "slots", "h", "hs", "y"):
        refused("null", name, a, **{p: None})
    refused("nsel", name, a, nsel=0)
    refused("max_tiles", name, a, max_tiles=0)
    refused("block_m", name, a, block_m=16)
    refused("H % 128", name, a, H=192)
    for p in ("x", "h", "y"):
        refused("16-byte", name, a, **{p: ODD})
    refused("4-byte", name, a, xs=P + 2)
    refused("too many tiles", name, a, max_tiles=1 << 22, I=768)
