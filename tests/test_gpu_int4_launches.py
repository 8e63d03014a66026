"""Every launch of the products with 4-bit matrices, each asked for by its sizes: tails of the K axis and
parts without a step, groups of every size with and without zero points, fp16 scales, inputs with a mean
far from 0, NaN rows, replays and two calls at once.  Bounds: test_gpu_int4.py."""
import pytest
import torch

from pdscope_amd import _lib, ops
from test_gpu_int4 import check, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16
REGISTERS, SPLIT, TILES_64, HALVES_128, TILES_128, TILES_256 = range(1, 7)


def takes(launch, T, N, K, G):
    assert _lib.load().pdscope_linear_int4_launch(T, N, K, G) == launch


CASES = [
    # x in registers: waves with two units, one and none behind the end; a last unit of 32, 64 or 96 inputs
    (REGISTERS, 13, 121_009, 1664, 128), (REGISTERS, 16, 121_009, 1664, 64), (REGISTERS, 14, 113_000, 1696, 32),
    (REGISTERS, 15, 112_385, 1792, 64), (REGISTERS, 16, 105_100, 1856, 64), (REGISTERS, 16, 105_001, 1920, 128),
    (REGISTERS, 16, 105_001, 1888, 32), (REGISTERS, 1, 131_089, 2048, 64), (REGISTERS, 8, 131_100, 1952, 32),
    (REGISTERS, 5, 140_003, 2048, 128),
    # few rows: four, two and one row tile a workgroup, 16 waves, one, two and four token tiles
    (SPLIT, 16, 98_300, 2048, 64), (SPLIT, 3, 70_001, 1696, 32), (SPLIT, 9, 8200, 96, 32), (SPLIT, 16, 4113, 2112, 64),
    (SPLIT, 4, 2050, 2208, 32), (SPLIT, 2, 4096, 4160, 64), (SPLIT, 11, 300, 1152, 128), (SPLIT, 20, 1003, 1056, 32),
    (SPLIT, 31, 4094, 2112, 64), (SPLIT, 48, 4001, 1408, 128),
    # 64 x 64 in four parts: fewer steps than parts, one more, the sums' buffers changed within the loop
    (TILES_64, 130, 4001, 128, 32), (TILES_64, 200, 3000, 640, 64), (TILES_64, 129, 4095, 2080, 32),
    (TILES_64, 250, 4096, 4096, 32), (TILES_64, 190, 2050, 4160, 64), (TILES_64, 255, 4001, 8192, 128),
    # 64 x 128 in two
    (HALVES_128, 500, 4001, 96, 32), (HALVES_128, 512, 4095, 384, 128), (HALVES_128, 449, 4096, 2112, 64),
    (HALVES_128, 511, 4002, 4096, 32), (HALVES_128, 512, 2049, 8192, 128),
    # 64 x 128
    (TILES_128, 1100, 4001, 128, 32), (TILES_128, 700, 4095, 2080, 32), (TILES_128, 1111, 4096, 2112, 64),
    (TILES_128, 1300, 4097, 4096, 128), (TILES_128, 2047, 4099, 2048, 64),
    # 64 x 256
    (TILES_256, 2048, 4096, 4096, 128), (TILES_256, 2000, 4050, 2080, 32), (TILES_256, 2047, 4095, 2112, 64),
    (TILES_256, 2048, 4001, 96, 32), (TILES_256, 1985, 4096, 192, 64), (TILES_256, 2048, 4089, 4192, 32)]


@pytest.mark.parametrize("launch,T,N,K,G", CASES)
@pytest.mark.parametrize("zeros,dtype,bias", [(False, BF16, True), (True, F16, False), (True, BF16, True)])
def test_products(launch, T, N, K, G, zeros, dtype, bias):
    takes(launch, T, N, K, G)
    codes, scales, z = make(N, K, G, zeros=zeros, dtype=dtype, seed=T)
    g = torch.Generator(device=DEV).manual_seed(N)
    x = torch.randn((T, K), generator=g, device=DEV).to(BF16)
    b = torch.randn(N, generator=g, device=DEV).to(BF16) if bias else None
    w = ops.int4_pack(codes, scales, z)
    y = ops.linear_int4(x, w, b)
    check(y, x, codes, scales, z, G, b)
    assert torch.equal(y, ops.linear_int4(x, w, b))


ONE_EACH = [(REGISTERS, 13, 121_009, 1664, 64), (REGISTERS, 2, 131_089, 2016, 32), (SPLIT, 16, 8300, 1056, 32),
            (SPLIT, 40, 1003, 1152, 128), (TILES_64, 200, 3001, 2080, 32), (HALVES_128, 500, 4001, 2112, 64),
            (TILES_128, 1100, 4001, 2176, 128), (TILES_256, 2000, 4095, 2112, 64)]


@pytest.mark.parametrize("launch,T,N,K,G", ONE_EACH)
def test_large_means_and_small_scales(launch, T, N, K, G):
    """fp16 scales (subnormal ones among them), inputs with a mean far from 0 and of 2^100."""
    takes(launch, T, N, K, G)
    codes, scales, z = make(N, K, G, zeros=True, dtype=F16, seed=9)
    scales[::3] *= 2.0 ** -10
    x = (torch.randn((T, K), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) + 30).to(BF16)
    w = ops.int4_pack(codes, scales, z)
    check(ops.linear_int4(x, w), x, codes, scales, z, G)
    x = (x * 2.0 ** 100).to(BF16)
    check(ops.linear_int4(x, w), x, codes, scales, z, G)


@pytest.mark.parametrize("launch,T,N,K,G", ONE_EACH)
def test_rows_outside_are_left_and_nan_rows_stay_their_own(launch, T, N, K, G):
    takes(launch, T, N, K, G)
    codes, scales, z = make(N, K, G, zeros=True, seed=4)
    w = ops.int4_pack(codes, scales, z)
    x = torch.randn((T, K), generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).to(BF16)
    room = torch.full((T + 4, N), 7.0, dtype=BF16, device=DEV)
    want = ops.linear_int4(x, w, out=room[2:T + 2]).clone()
    assert (room[:2] == 7).all() and (room[T + 2:] == 7).all()
    x[T // 2, 5], x[T - 1, K - 1] = float("nan"), float("inf")
    y = ops.linear_int4(x, w)
    assert torch.isnan(y[T // 2]).all() and torch.isnan(y[T - 1]).all()
    keep = torch.ones(T, dtype=torch.bool, device=DEV)
    keep[T // 2] = keep[T - 1] = False
    assert torch.equal(y[keep], want[keep])


@pytest.mark.parametrize("launch,T,N,K,G", ONE_EACH)
def test_replays_and_two_calls_at_once(launch, T, N, K, G):
    takes(launch, T, N, K, G)
    w = [ops.int4_pack(*make(N, K, G, zeros=True, seed=s)) for s in (6, 7)]
    x = torch.randn((T, K), generator=torch.Generator(device=DEV).manual_seed(8), device=DEV).to(BF16)
    want = [ops.linear_int4(x, m) for m in w]
    streams = [torch.cuda.Stream() for _ in w]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        got = []
        for s, m in zip(streams, w):
            with torch.cuda.stream(s):
                got.append(ops.linear_int4(x, m))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [ops.linear_int4(x, m) for m in w]
    for _ in range(3):
        for y in got:
            y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
