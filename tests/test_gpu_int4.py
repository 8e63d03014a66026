"""4-bit matrices with group scales: layout, quantising and the products of 1 to a few thousand rows.

The product's bound, with u = 2^-24: q x is exact, a group's two sums are off by (G + 2) u of their
summed magnitudes, and what is made of them by 3 roundings a group, one for each addition to the
total (two a group where the zero points' part is taken off by itself) and one for each of up to 16
parts of the K axis: (G + 2 K / G + 24) u (s (q + z) . |x|), then half a step of bf16."""
import pytest
import torch

from moe64 import assert_within
from pdscope_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16
U, B = 2.0 ** -24, 2.0 ** -8


def make(N, K, G, *, zeros=False, dtype=BF16, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = (0.002 + 0.01 * torch.rand((N, K // G), generator=g, device=DEV)).to(dtype)
    z = torch.randint(0, 16, (N, K // G), generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return codes, scales, z


def values64(codes, scales, z, G):
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(1).double()
    z = torch.full_like(scales, 8.0, dtype=torch.float64) if z is None else z.double()
    s = scales.double().repeat_interleave(G, 1)
    z = z.repeat_interleave(G, 1)
    return (q - z) * s, (q + z) * s.abs()


def check(y, x, codes, scales, z, G, bias=None):
    w, mass = values64(codes, scales, z, G)
    K = x.shape[1]
    want = x.double() @ w.T
    bound = (G + 2 * K // G + 24) * U * (x.double().abs() @ mass.T)
    if bias is not None:
        want, bound = want + bias.double(), bound + 2 * U * bias.double().abs()
    assert_within(y, want, (1 + B) * bound + B * want.abs() + 2.0 ** -133)


@pytest.mark.parametrize("N,K,G", [(1, 32, 32), (16, 128, 128), (17, 160, 32), (5, 192, 64), (100, 2048, 128), (33, 4096, 64),
                                   (250, 96, 32)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_layout_round_trip(N, K, G, zeros, dtype):
    codes, scales, z = make(N, K, G, zeros=zeros, dtype=dtype, seed=N + K)
    w = ops.int4_pack(codes, scales, z)
    assert (w.N, w.K, w.group, w.zeros, w.scale_dtype) == (N, K, G, zeros, dtype)
    assert w.units.numel() == ops.int4_bytes(N, K, G, zeros)
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(1).float()
    zf = 8.0 if z is None else z.float().repeat_interleave(G, 1)
    assert torch.equal(ops.int4_dequantize(w), ((q - zf) * scales.float().repeat_interleave(G, 1)).to(BF16))


@pytest.mark.parametrize("N,K,G", [(1, 32, 32), (31, 2048, 128), (64, 4096, 64), (77, 224, 32), (4096, 2048, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantise(N, K, G, zeros):
    """The stated rule in torch's fp32, whose products, quotients and roundings are the same ones."""
    g = torch.Generator(device=DEV).manual_seed(N)
    weight = (0.02 * torch.randn((N, K), generator=g, device=DEV) + 0.01).to(BF16)
    weight[0, :32] = 0
    if N > 1:
        weight[1] = 0.25
    v = weight.float().unflatten(1, (-1, G))
    if zeros:
        lo, hi = (-v).amax(2).clamp(min=0), v.amax(2).clamp(min=0)
        s = ((hi + lo) / 15).to(BF16).float()
        z = torch.where(s > 0, torch.round(lo / s).clamp(max=15), torch.zeros_like(s))
    else:
        s = (v.abs().amax(2) / 7).to(BF16).float()
        z = torch.full_like(s, 8.0)
    q = torch.where(s.unsqueeze(2) > 0, torch.round(v / s.unsqueeze(2)) + z.unsqueeze(2), z.unsqueeze(2)).clamp(0, 15)
    w = ops.int4_quantize(weight, G, zeros)
    q = q.flatten(1).to(torch.uint8)
    want = ops.int4_pack(q[:, 0::2] | (q[:, 1::2] << 4), s.to(BF16), z.to(torch.uint8) if zeros else None)
    assert torch.equal(w.units, want.units)
    # and near the matrix: half a step, two roundings of the scale's eight bits over 15 steps
    step = s.repeat_interleave(G, 1)
    assert ((ops.int4_dequantize(w).float() - weight.float()).abs() <= 0.5 * step + 0.14 * step + 2.0 ** -8 * weight.float().abs()).all()


SIZES = [(1, 1, 32, 32), (1, 16, 128, 128), (2, 15, 64, 64), (1, 4096, 2048, 128), (3, 513, 4096, 64), (5, 4097, 2816, 32),
         (15, 33, 96, 32), (16, 2048, 4096, 128), (17, 100, 352, 32), (31, 257, 768, 128), (33, 640, 1408, 128),
         (48, 255, 2048, 64), (64, 1000, 1024, 32), (65, 129, 256, 64), (128, 512, 2048, 128), (200, 77, 160, 32),
         (513, 384, 640, 128), (1031, 1100, 2048, 64), (2048, 256, 4096, 128),
         # the launch for many rows: one step of the K axis, two, odd ones, ragged edges of every kind
         (800, 1000, 96, 32), (800, 1000, 128, 128), (3100, 257, 352, 32), (3071, 255, 192, 64), (1500, 520, 1408, 128),
         (1025, 771, 4096, 64), (2049, 513, 1056, 32),
         # smaller tiles, whose steps two halves of a workgroup share: one step, an odd count of them
         (70, 2100, 128, 128), (200, 1030, 1056, 32), (130, 4100, 640, 64), (513, 2048, 4096, 128), (512, 4095, 352, 32),
         (449, 4096, 128, 64), (700, 1500, 2048, 128), (24, 16384, 1408, 128),
         # tiles of 128 rows without parts: one step, an odd count of them, ragged edges
         (700, 4000, 128, 64), (1300, 4097, 352, 32), (650, 3900, 1408, 128), (1111, 2500, 2048, 32),
         (2048, 4097, 160, 32), (2500, 4100, 256, 128), (1800, 2222, 192, 64), (1601, 4098, 128, 32),
         # many row tiles for one workgroup
         (1, 20000, 2048, 128), (3, 16401, 1152, 32), (16, 33000, 1984, 64), (2, 9000, 8192, 128), (4, 5000, 4096, 128),
         (1, 70000, 2048, 128), (9, 66001, 2016, 32), (16, 80000, 1984, 64), (2, 5000, 352, 32), (13, 8193, 1088, 64), (16, 4113, 96, 32)]


@pytest.mark.parametrize("T,N,K,G", SIZES)
@pytest.mark.parametrize("zeros,bias", [(False, False), (True, True)])
def test_products(T, N, K, G, zeros, bias):
    codes, scales, z = make(N, K, G, zeros=zeros, seed=T)
    g = torch.Generator(device=DEV).manual_seed(N)
    x = torch.randn((T, K), generator=g, device=DEV).to(BF16)
    b = torch.randn(N, generator=g, device=DEV).to(BF16) if bias else None
    w = ops.int4_pack(codes, scales, z)
    y = ops.linear_int4(x, w, b)
    check(y, x, codes, scales, z, G, b)
    assert torch.equal(y, ops.linear_int4(x, w, b))


@pytest.mark.parametrize("T", [1, 7, 40, 300, 3100])
def test_fp16_scales_and_large_inputs(T):
    """fp16 scales (subnormal ones among them), inputs with a mean far from 0 and of 2^100."""
    N, K, G = 200, 1024, 64
    codes, scales, z = make(N, K, G, zeros=True, dtype=F16, seed=9)
    scales[::3] *= 2.0 ** -10
    x = (torch.randn((T, K), device=DEV) + 30).to(BF16)
    w = ops.int4_pack(codes, scales, z)
    check(ops.linear_int4(x, w), x, codes, scales, z, G)
    x = (x * 2.0 ** 100).to(BF16)
    check(ops.linear_int4(x, w), x, codes, scales, z, G)


def test_every_count_of_rows():
    N, K, G = 80, 256, 32
    codes, scales, z = make(N, K, G, seed=3)
    w = ops.int4_pack(codes, scales)
    x = torch.randn((150, K), device=DEV).to(BF16)
    for T in list(range(1, 70)) + [79, 80, 81, 95, 96, 97, 127, 128, 129, 150]:
        check(ops.linear_int4(x[:T], w), x[:T], codes, scales, z, G)


@pytest.mark.parametrize("T", [3, 40, 200, 3100])
def test_rows_outside_are_left_and_nan_rows_stay_their_own(T):
    N, K, G = 100, 160, 32
    codes, scales, z = make(N, K, G, zeros=True, seed=4)
    w = ops.int4_pack(codes, scales, z)
    x = torch.randn((T, K), device=DEV).to(BF16)
    room = torch.full((T + 4, N), 7.0, dtype=BF16, device=DEV)
    want = ops.linear_int4(x, w, out=room[2:T + 2]).clone()
    assert (room[:2] == 7).all() and (room[T + 2:] == 7).all()
    x[1, 5], x[T - 1, K - 1] = float("nan"), float("inf")
    y = ops.linear_int4(x, w)
    assert torch.isnan(y[1]).all() and torch.isnan(y[T - 1]).all()
    keep = torch.ones(T, dtype=torch.bool, device=DEV)
    keep[1] = keep[T - 1] = False
    assert torch.equal(y[keep], want[keep])


def test_a_matrix_past_2_to_the_31_bytes():
    N, K, G = 2_200_000, 2048, 128
    codes = torch.randint(0, 256, (64, K // 2), device=DEV, dtype=torch.uint8).repeat(N // 64 + 1, 1)[:N]
    scales = torch.linspace(0.001, 0.01, N, device=DEV).to(BF16).unsqueeze(1).expand(N, K // G).contiguous()
    w = ops.int4_pack(codes, scales)
    assert w.units.numel() > 2 ** 31
    for T in (2, 70):
        x = torch.randn((T, K), device=DEV).to(BF16)
        y = ops.linear_int4(x, w)
        for a in (0, N // 2 // 16 * 16, N - 100):
            check(y[:, a:a + 100].contiguous(), x, codes[a:a + 100], scales[a:a + 100], None, G)


@pytest.mark.parametrize("T", [1, 20, 60, 200, 900, 2300])
def test_outputs_at_addresses_that_16_bytes_do_not_divide(T):
    N, K, G = 1040, 384, 128
    codes, scales, z = make(N, K, G, zeros=True, seed=12)
    w = ops.int4_pack(codes, scales, z)
    x = torch.randn((T, K), device=DEV).to(BF16)
    want = ops.linear_int4(x, w)
    for off in (1, 2, 4):
        room = torch.full((T * N + 16,), 7.0, dtype=BF16, device=DEV)
        ops.linear_int4(x, w, out=room[off:off + T * N].view(T, N))
        assert torch.equal(room[off:off + T * N].view(T, N), want)
        assert (room[:off] == 7).all() and (room[off + T * N:] == 7).all()
    check(want, x, codes, scales, z, G)


def test_more_than_2_to_the_31_outputs():
    T, N, K, G = 16_400, 140_000, 64, 64
    codes, scales, _ = make(N, K, G, seed=11)
    w = ops.int4_pack(codes, scales)
    x = torch.randn((T, K), device=DEV).to(BF16)
    y = ops.linear_int4(x, w)
    rows = torch.tensor([0, 63, 64, T // 2, T - 1], device=DEV)
    check(y[rows], x[rows], codes, scales, None, G)
    for at in (0, N - 3):
        check(y[:, at:at + 3].contiguous(), x, codes[at:at + 3], scales[at:at + 3], None, G)


@pytest.mark.parametrize("T", [2, 40, 1700])
def test_replay_and_another_stream(T):
    N, K, G = 300, 2048, 128
    codes, scales, z = make(N, K, G, zeros=True, seed=5)
    w = ops.int4_pack(codes, scales, z)
    x = torch.randn((T, K), device=DEV).to(BF16)
    want = ops.linear_int4(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_int4(x, w)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_int4(x, w)
    for _ in range(3):
        got.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_two_streams_at_once():
    """Two calls of the launch for many rows that may run together: nothing is shared."""
    T, N, K, G = 1000, 900, 512, 64
    w = [ops.int4_pack(*make(N, K, G, zeros=True, seed=s)) for s in (6, 7)]
    x = torch.randn((T, K), device=DEV).to(BF16)
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
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_no_rows():
    codes, scales, _ = make(48, 64, 32)
    w = ops.int4_pack(codes, scales)
    assert ops.linear_int4(torch.empty((0, 64), dtype=BF16, device=DEV), w).shape == (0, 48)


def test_refusals():
    codes, scales, z = make(48, 256, 64, zeros=True)
    with pytest.raises(ValueError, match="groups of 32"):
        ops.int4_pack(codes, scales[:, :1].contiguous())
    with pytest.raises(ValueError, match="scales must be"):
        ops.int4_pack(codes, scales[:20].contiguous())
    with pytest.raises(ValueError, match="bf16 or fp16"):
        ops.int4_pack(codes, scales.float())
    with pytest.raises(ValueError, match="zeros must be"):
        ops.int4_pack(codes, scales, z[:, :2].contiguous())
    w = ops.int4_pack(codes, scales, z)
    x = torch.zeros((3, 256), dtype=BF16, device=DEV)
    with pytest.raises(ValueError, match="x must be"):
        ops.linear_int4(x[:, :128].contiguous(), w)
    with pytest.raises(ValueError, match="bias must be"):
        ops.linear_int4(x, w, torch.zeros(47, dtype=BF16, device=DEV))
    with pytest.raises(ValueError, match="out must be"):
        ops.linear_int4(x, w, out=torch.zeros((3, 49), dtype=BF16, device=DEV))
    with pytest.raises(ValueError, match="size of its shape"):
        ops.linear_int4(x, ops.Int4Weight(w.units, 64, 256, 64, True))
    with pytest.raises(ValueError, match="16-byte"):
        room = torch.zeros(3 * 256 + 1, dtype=BF16, device=DEV)
        ops.linear_int4(room[1:].view(3, 256), w)
    with pytest.raises(ValueError, match="contiguous"):
        ops.linear_int4(torch.zeros((3, 512), dtype=BF16, device=DEV)[:, ::2], w)


# ------------------------------------------------------- a model's linear modules

def small_model(seed=1):
    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM
    cfg = Qwen3MoeConfig(vocab_size=331, hidden_size=256, intermediate_size=512, moe_intermediate_size=128,
                         num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                         num_experts=32, num_experts_per_tok=4, norm_topk_prob=True, decoder_sparse_step=1,
                         mlp_only_layers=[], initializer_range=0.05)
    torch.manual_seed(seed)
    model = Qwen3MoeForCausalLM(cfg).to(BF16).eval()
    with torch.no_grad():
        for d in model.model.layers:
            d.mlp.gate.weight.normal_(0.0, 0.5)
    return cfg, model


PROJECTIONS = [f"model.layers.{layer}.self_attn.{p}_proj" for layer in (0, 1) for p in "qkvo"]


def test_modules_of_a_model():
    """Every linear module outside the expert blocks is replaced and gives its own 4-bit matrix'
    products; routers, experts and what is kept are as they were."""
    from pdscope_amd.hf import Int4Linear, install_int4_linears
    _, model = small_model()
    model.to(DEV)
    before = {n: m for n, m in model.named_modules() if isinstance(m, torch.nn.Linear)}
    names = install_int4_linears(model, 64, zeros=True, keep=("lm_head",))
    assert sorted(names) == sorted(PROJECTIONS)
    after = dict(model.named_modules())
    for n, m in before.items():
        assert (type(after[n]) is Int4Linear) == (n in names) and (n in names or after[n] is m)
    for n in names:
        q, m = after[n], before[n]
        for shape in ((1, 1), (3, 7), (2, 80)):
            x = torch.randn((*shape, m.in_features), device=DEV).to(BF16)
            w = ops.int4_dequantize(ops.int4_quantize(m.weight.detach(), 64, True)).double()
            y = q(x)
            want = x.double() @ w.T
            # the dequantised matrix is rounded to bf16: half a step of each weight more than the sums' bound
            bound = (64 + 256 // 64 + 24) * U * 32 * (x.double().abs() @ w.abs().T) + B * (x.double().abs() @ w.abs().T)
            assert y.shape == (*shape, m.out_features) and y.dtype is BF16
            assert_within(y, want, (1 + B) * bound + B * want.abs() + 2.0 ** -133)
    x = torch.randn((2, 256), device=DEV).to(BF16).requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        after[names[0]](x)
    with pytest.raises(ValueError, match="whole groups"):
        install_int4_linears(torch.nn.Sequential(torch.nn.Linear(96, 8)).to(BF16).to(DEV), 64)
    with pytest.raises(ValueError, match="bf16 on the GPU"):
        install_int4_linears(torch.nn.Sequential(torch.nn.Linear(128, 8)), 64)


def test_model_session_on_four_bit_linears():
    """A prompt and two tokens through a session with 4-bit projections and head against the same
    model with these modules' dequantised matrices in bf16: they differ by the roundings of bf16
    matrices and of attention, as the two models of test_gpu_hybrid.py do."""
    from pdscope_amd.hf import Int4Linear, ModelSession
    cfg, ours = small_model()
    _, native = small_model()
    native.to(DEV)
    with torch.no_grad():
        for n, m in native.named_modules():
            if n in PROJECTIONS or n == "lm_head":
                m.weight.copy_(ops.int4_dequantize(ops.int4_quantize(m.weight.detach(), 128)))
    session = ModelSession(ours, hot_per_layer=6, speculative_slots=2, demand_slots=2, device=0, int4_group=128)
    try:
        assert sorted(session.int4_linears) == sorted(PROJECTIONS + ["lm_head"])
        assert type(ours.lm_head) is Int4Linear
        ids = torch.randint(0, cfg.vocab_size, (1, 24), generator=torch.Generator().manual_seed(2)).to(DEV)
        with torch.no_grad():
            past_a = past_b = None
            for step in range(3):
                session.step = step
                a = native(ids, past_key_values=past_a, use_cache=True)
                b = ours(ids, past_key_values=past_b, use_cache=True)
                past_a, past_b = a.past_key_values, b.past_key_values
                r, g = a.logits[0, -1].float(), b.logits[0, -1].float()
                assert (r - g).norm() <= 3e-2 * r.norm()
                ids = r.argmax().view(1, 1)
    finally:
        session.close()
