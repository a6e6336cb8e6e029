"""4-bit expert weights on the GPU against plain 64-bit implementations.

Two kinds of checks. Exact ones: activations are small integers and scales
powers of two, so every product and every partial sum is a multiple of 1/4
below 2^22 in magnitude and fp32 holds it exactly in any order; the output then
has to equal the 64-bit result rounded once. Bounded ones: random data, each
output within a bound that counts roundings,

    half a step of the output's type, u = eps / 2, relative to the value,
    u for each weight that a kernel rounds to the activations' type,
    fp32 sums of K terms: 2 K 2^-24 of the sum of their magnitudes
"""
import pytest

torch = pytest.importorskip("torch")

import mail_b200 as mb  # noqa: E402
from mail_b200 import _lib, int4  # noqa: E402

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
DEV = "cuda"


@pytest.fixture(params=["rows", "tiles"])
def kernel(request):
    """Each test with the row kernels and with the tensor-core tiles."""
    lib = _lib.load()
    before = lib.moe_get_option(_lib.OPT_INT4_GEMM)
    assert lib.moe_set_option(_lib.OPT_INT4_GEMM, int(request.param == "tiles")) == 0
    yield request.param
    assert mb.device_error() == 0
    assert lib.moe_set_option(_lib.OPT_INT4_GEMM, before) == 0


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def weights(E, N, K, group, dtype, seed, exact=False):
    """Packed 4-bit weights as logical (E, K, N), scales, 64-bit values [E, N, K]."""
    g = gen(seed)
    q = torch.randint(0, 16, (E, N, K), device=DEV, generator=g)
    packed = (q[..., 0::2] | (q[..., 1::2] << 4)).to(torch.uint8)
    if exact:
        s = torch.tensor([0.25, 0.5, 1.0], device=DEV)[torch.randint(0, 3, (E, N, K // group), device=DEV, generator=g)]
    else:
        s = (torch.rand((E, N, K // group), device=DEV, generator=g) + 0.5) * 0.3 / K ** 0.5
    s = s.to(dtype)
    wide = (q.double() - 8) * s.double().repeat_interleave(group, dim=2)
    return packed.transpose(1, 2), s, wide


def small_ints(shape, dtype, seed):
    return torch.randint(-2, 3, shape, device=DEV, generator=gen(seed)).to(dtype)


def routing(T, E, k, seed):
    g = gen(seed)
    w, ids = torch.topk(torch.rand((T, E), device=DEV, generator=g), k, dim=1)
    return torch.softmax(w, dim=1).float(), ids.to(torch.int32)


def grouped_ref(x, wide, sizes):
    out = torch.zeros((x.shape[0], wide.shape[1]), dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(out)
    r = 0
    for e, n in enumerate(sizes):
        n = min(n, x.shape[0] - r)
        out[r:r + n] = x[r:r + n].double() @ wide[e].t()
        mag[r:r + n] = x[r:r + n].double().abs() @ wide[e].abs().t()
        r += n
    return out, mag


def layer_ref(x, w13, w2, wts, ids, dtype):
    """(y, bound of |kernel - y| before the output's rounding) in 64 bits."""
    u = half_step(dtype)
    T, H = x.shape
    E, two_i, _ = w13.shape
    I = two_i // 2
    y = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(y)
    f1, f2 = u + 2 * H * 2.0 ** -24, u + 2 * I * 2.0 ** -24
    for e in range(E):
        tok, col = torch.nonzero(ids == e, as_tuple=True)
        if tok.numel() == 0:
            continue
        r = x[tok].double()
        gu, ga = r @ w13[e].t(), r.abs() @ w13[e].abs().t()
        g, up = gu[:, :I], gu[:, I:]
        silu = g * torch.sigmoid(g)
        h = silu * up
        # |silu'| <= 1.1; the fast exponential and quotient: 2^-18 relative is
        # several of their documented steps for |g| < 64; h's own rounding u,
        # and half of the smallest number of its type
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        dh = 1.1 * up.abs() * f1 * ga[:, :I] + (silu.abs() + 1.1 * f1 * ga[:, :I]) * f1 * ga[:, I:] \
            + (u + 2.0 ** -18) * h.abs() + tiny
        p = wts[tok, col].double().unsqueeze(1)
        y.index_add_(0, tok, p * (h @ w2[e].t()))
        bound.index_add_(0, tok, p.abs() * ((dh + f2 * (h.abs() + dh)) @ w2[e].abs().t()))
    k = ids.shape[1]
    return y, bound * (1 + 2 * k * 2.0 ** -24)


def assert_within(out, ref, bound, dtype):
    u = half_step(dtype)
    lim = bound + u * (ref.abs() + bound) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    over = (out.double() - ref).abs() - lim
    assert bool((over <= 0).all()), f"worst excess {float(over.max()):.3e}"


# ------------------------------------------------------- quantising, reading back


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("wdtype,sdtype", [(BF, BF), (HF, HF), (torch.float32, BF), (torch.float32, HF), (BF, HF),
                                           (HF, BF)])
@pytest.mark.parametrize("R,C", [(1, 128), (3, 384), (257, 640), (1000, 2048)])
def test_quant_is_the_exact_quotient(group, wdtype, sdtype, R, C):
    w = (torch.randn((R, C), device=DEV, generator=gen(R)) * 0.02).to(wdtype)
    w[0, :group] = 0  # a group of zeros
    # values on the borders between two steps: multiples of half a step
    w[-1, -group:] = (torch.arange(group, device=DEV) % 15 - 7).to(wdtype) / 2
    w[-1, -1] = 7.0
    q, s = mb.quant_int4_groups(w, group, scale_dtype=sdtype)
    wd = w.double().view(R, C // group, group)
    amax = wd.abs().amax(-1)
    s_ref = (amax / 7).float().to(sdtype)
    assert torch.equal(s, s_ref)
    sd = s_ref.double().unsqueeze(-1)
    steps = torch.where(sd > 0, wd / sd.clamp_min(1e-300), torch.zeros_like(wd)).round().clamp(-8, 7) + 8
    got = torch.stack((q & 15, q >> 4), dim=-1).view(R, C // group, group)
    assert torch.equal(got.double(), steps)
    for dt in (BF, HF, torch.float32):
        vals = mb.dequant_int4_groups(q, s, dtype=dt)
        # 4-bit steps times a 16-bit scale are exact in fp32: one rounding to dt
        assert torch.equal(vals, ((steps - 8) * sd).float().to(dt).view(R, C))


def test_quant_marks_groups_that_are_not_finite():
    w = torch.randn((4, 256), device=DEV, generator=gen(0))
    w[0, 3] = float("nan")
    w[1, 130] = float("inf")
    w[2, 255] = -float("inf")
    w[3, 64] = 7.5 * 65504  # absmax / 7 is beyond fp16, not beyond bf16
    for sdtype, bad in ((BF, {(0, 0), (1, 1), (2, 1)}), (HF, {(0, 0), (1, 1), (2, 1), (3, 0)})):
        q, s = mb.quant_int4_groups(w, 128, scale_dtype=sdtype)
        assert {tuple(i) for i in torch.isnan(s).nonzero().tolist()} == bad
        vals = mb.dequant_int4_groups(q, s, dtype=torch.float32).view(4, 2, 128)
        for r in range(4):
            for c in range(2):
                assert bool(torch.isnan(vals[r, c]).all()) == ((r, c) in bad)


def test_quant_takes_strided_weights_and_leaves_them():
    w = torch.randn((64, 512), device=DEV, generator=gen(1)).to(BF)
    keep = w.clone()
    q, s = mb.quant_int4_groups(w[::2, 128:384], 64)
    q2, s2 = mb.quant_int4_groups(w[::2, 128:384].contiguous(), 64)
    assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(w, keep)
    e, se = mb.quant_int4_groups(w[:0], 64)
    assert e.shape == (0, 256) and se.shape == (0, 8)


# --------------------------------------------------------------- grouped products


GROUPED = [
    # K, N, group, sizes
    (32, 1, 32, [1]),
    (128, 16, 128, [0, 1, 0]),
    (128, 17, 64, [2, 0, 7, 1]),
    (96, 33, 32, [5]),
    (256, 40, 128, [8, 9, 16, 17]),
    (1056, 101, 32, [0, 33, 64, 1, 0]),
    (448, 130, 64, [129, 3]),
    (640, 250, 128, [31, 300, 0, 70]),
    (2048, 1536, 128, [1] * 8 + [0] * 24),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("K,N,group,sizes", GROUPED)
def test_grouped_matmul_exact(dtype, K, N, group, sizes, kernel):
    E, T = len(sizes), sum(sizes)
    w, s, wide = weights(E, N, K, group, dtype, K + N, exact=True)
    x = small_ints((T, K), dtype, T)
    ref, mag = grouped_ref(x, wide, sizes)
    assert float(mag.max()) * 4 < 2 ** 24
    out = mb.grouped_matmul_int4(x, w, s, torch.tensor(sizes, dtype=torch.int32, device=DEV))
    assert out.dtype == dtype and torch.equal(out, ref.to(dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("K,N,group,sizes", GROUPED)
def test_grouped_matmul_random(dtype, K, N, group, sizes, kernel):
    E, T = len(sizes), sum(sizes)
    w, s, wide = weights(E, N, K, group, dtype, K)
    x = torch.randn((T, K), device=DEV, generator=gen(N)).to(dtype)
    ref, mag = grouped_ref(x, wide, sizes)
    out = mb.grouped_matmul_int4(x, w, s, torch.tensor(sizes, device=DEV))
    assert_within(out, ref, (half_step(dtype) + 2 * K * 2.0 ** -24) * mag, dtype)


@pytest.mark.parametrize("sizes", [[3, 0, 2], [0, 0, 0], [4, 4, 40], [-3, 5, 0], [12, 0, 0], [12, 5, 7], [40, 0, 9],
                                   [0, 13, 1]])
def test_grouped_matmul_sizes_that_do_not_add_up(sizes, kernel):
    """Rows behind the last group are zero; counts past the rows are cut off;
    negative counts are empty groups."""
    T, K, N = 12, 128, 50
    w, s, wide = weights(3, N, K, 128, BF, 5, exact=True)
    x = small_ints((T, K), BF, 3)
    ref, _ = grouped_ref(x, wide, [max(n, 0) for n in sizes])
    for dt in (torch.int32, torch.int64):
        out = mb.grouped_matmul_int4(x, w, s, torch.tensor(sizes, dtype=dt, device=DEV))
        assert torch.equal(out, ref.to(BF))
    out = mb.grouped_matmul_int4(x[:0], w, s, torch.tensor([0, 0, 0], device=DEV))
    assert out.shape == (0, N)


def test_grouped_matmul_many_experts_and_offsets(kernel):
    E, K, N = 1024, 64, 24
    sizes = torch.randint(0, 4, (E,), device=DEV, generator=gen(2))
    w, s, wide = weights(E, N, K, 32, HF, 1, exact=True)
    x = small_ints((int(sizes.sum()), K), HF, 9)
    ref, _ = grouped_ref(x, wide, sizes.tolist())
    assert torch.equal(mb.grouped_matmul_int4(x, w, s, sizes), ref.to(HF))


def test_grouped_matmul_weights_past_32_bit_offsets(kernel):
    """The last expert's weights lie behind 2^32 nibbles."""
    E, K, N = 9, 7168, 65536 + 8192
    assert E * K * N > 2 ** 32
    packed = torch.zeros((E, N, K // 2), dtype=torch.uint8, device=DEV)
    packed[-1] = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=DEV, generator=gen(0))
    s = torch.ones((E, N, K // 128), dtype=BF, device=DEV)
    x = small_ints((2, K), BF, 1)
    sizes = torch.tensor([0] * (E - 1) + [2], device=DEV)
    q = torch.stack((packed[-1] & 15, packed[-1] >> 4), dim=-1).view(N, K)
    ref = torch.empty((2, N), dtype=torch.float64, device=DEV)
    for n in range(0, N, 8192):
        ref[:, n:n + 8192] = x.double() @ (q[n:n + 8192].double() - 8).t()
    assert torch.equal(mb.grouped_matmul_int4(x, packed.transpose(1, 2), s, sizes), ref.to(BF))


@pytest.mark.parametrize("dtype,E,K,N,group,sizes", [
    (BF, 2, 4096, 36864, 128, [0, 2]), (BF, 2, 4096, 36864, 32, [3, 0]), (HF, 16, 2048, 6144 + 130, 64, [20] * 16),
    (BF, 3, 4096, 16384, 128, [700, 1, 600]), (HF, 3, 4096, 16384, 32, [700, 1, 600]),
    (BF, 3, 4096, 16384, 64, [300, 256, 600])])
def test_grouped_matmul_long_pipelines(dtype, E, K, N, group, sizes, kernel):
    """Many tiles of many blocks for each CTA, again and again: a stage that is
    refilled while it is read shows here."""
    w, s, wide = weights(E, N, K, group, dtype, 7, exact=True)
    x = small_ints((sum(sizes), K), dtype, 8)
    ref = grouped_ref(x, wide, sizes)[0].to(dtype)
    gs = torch.tensor(sizes, device=DEV)
    for _ in range(10 if kernel == "tiles" else 2):
        assert torch.equal(mb.grouped_matmul_int4(x, w, s, gs), ref)


def test_grouped_matmul_strided_inputs_and_other_layouts(kernel):
    w, s, wide = weights(3, 48, 256, 64, BF, 5, exact=True)
    sizes = torch.tensor([2, 0, 3], device=DEV)
    big = small_ints((10, 512), BF, 3)
    x = big[::2, 128:384]
    ref, _ = grouped_ref(x, wide, [2, 0, 3])
    assert torch.equal(mb.grouped_matmul_int4(x, w, s, sizes), ref.to(BF))
    # weights whose storage is not K-major are copied, with a warning once
    other = w.contiguous()
    assert torch.equal(mb.grouped_matmul_int4(x, other, s, sizes), ref.to(BF))
    every = torch.tensor([2, 9, 0, 9, 3, 9], device=DEV)[::2]
    assert torch.equal(mb.grouped_matmul_int4(x, w, s, every), ref.to(BF))


def test_grouped_matmul_keeps_nan_and_inf_to_their_rows(kernel):
    w, s, wide = weights(2, 64, 256, 128, BF, 5, exact=True)
    x = small_ints((20, 256), BF, 3)
    ref, _ = grouped_ref(x, wide, [9, 11])
    x[4, 17] = float("nan")
    x[15, 200] = float("inf")
    out = mb.grouped_matmul_int4(x, w, s, torch.tensor([9, 11], device=DEV))
    rows = [r for r in range(20) if r not in (4, 15)]
    assert torch.equal(out[rows], ref.to(BF)[rows])
    assert bool(torch.isnan(out[4]).all())
    assert not bool(torch.isfinite(out[15]).any() and (wide[1, :, 200] != 0).all())


# ---------------------------------------------------------------------- the layer


LAYER = [
    # T, E, k, H, I, group
    (1, 4, 1, 32, 32, 32),
    (1, 128, 8, 256, 96, 32),
    (2, 8, 2, 384, 640, 128),
    (5, 3, 3, 192, 128, 64),
    (16, 64, 8, 256, 128, 64),
    (33, 8, 4, 512, 256, 128),
    (130, 16, 8, 256, 128, 128),
    (300, 4, 2, 320, 160, 32),
    (520, 5, 3, 256, 384, 128),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,E,k,H,I,group", LAYER)
def test_layer(dtype, T, E, k, H, I, group, kernel):
    w13, s13, wide13 = weights(E, 2 * I, H, group, dtype, 1)
    w2, s2, wide2 = weights(E, H, I, group, dtype, 2)
    x = torch.randn((T, H), device=DEV, generator=gen(3)).to(dtype)
    wts, ids = routing(T, E, k, 4)
    ref, bound = layer_ref(x, wide13, wide2, wts, ids, dtype)
    y = mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2))
    assert y.dtype == dtype
    assert_within(y, ref, bound, dtype)
    assert torch.equal(y, mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2)))
    assert mb.device_error() == 0


@pytest.mark.parametrize("T", [3, 40, 700])
def test_layer_slots_that_name_no_expert(T, kernel):
    """Ids outside [0, E) add nothing, a token without any gives zeros, an
    expert named twice by one token counts twice."""
    E, k, H, I = 6, 4, 256, 128
    w13, s13, wide13 = weights(E, 2 * I, H, 128, BF, 1)
    w2, s2, wide2 = weights(E, H, I, 128, BF, 2)
    x = torch.randn((T, H), device=DEV, generator=gen(3)).to(BF)
    ids = torch.randint(-1, E + 1, (T, k), device=DEV, generator=gen(5)).to(torch.int32)
    ids[0] = -1
    ids[1] = 2
    wts = torch.randn((T, k), device=DEV, generator=gen(6))
    ref, bound = layer_ref(x, wide13, wide2, wts, ids, BF)
    y = mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2))
    assert bool((y[0] == 0).all())
    assert_within(y, ref, bound, BF)


@pytest.mark.parametrize("T", [2, 130, 600])
def test_layer_from_logits_matches_router_and_layer(T, kernel):
    E, k, H, I = 16, 4, 256, 128
    w13, s13, _ = weights(E, 2 * I, H, 64, BF, 1)
    w2, s2, _ = weights(E, H, I, 64, BF, 2)
    x = torch.randn((T, H), device=DEV, generator=gen(3)).to(BF)
    logits = torch.randn((T, E), device=DEV, generator=gen(4))
    y, wts, ids = mb.fused_moe_mlp_from_logits(x, w13, w2, logits, k, scoring="sigmoid", scales=(s13, s2))
    ids2, wts2 = mb.route_topk(logits, k, scoring="sigmoid")
    assert torch.equal(ids, ids2) and torch.equal(wts, wts2)
    assert torch.equal(y, mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2)))


@pytest.mark.parametrize("sizes", [[1, 0, 0], [3, 9, 0], [40, 0, 77], [200, 300, 140]])
def test_pre_routed_layer(sizes, kernel):
    E, H, I, dtype = 3, 256, 192, HF
    w13, s13, wide13 = weights(E, 2 * I, H, 64, dtype, 1)
    w2, s2, wide2 = weights(E, H, I, 64, dtype, 2)
    T = sum(sizes) + 2
    x = torch.randn((T, H), device=DEV, generator=gen(3)).to(dtype)
    ids = torch.repeat_interleave(torch.arange(E, device=DEV), torch.tensor(sizes, device=DEV))
    ids = torch.cat((ids, torch.tensor([-1, -1], device=DEV))).view(T, 1)
    ref, bound = layer_ref(x, wide13, wide2, torch.ones((T, 1), device=DEV), ids, dtype)
    out = mb.fused_moe_mlp(x, w13, w2, torch.tensor(sizes, device=DEV), scales=(s13, s2))
    assert bool((out[-2:] == 0).all())
    assert_within(out, ref, bound, dtype)


def test_quantise_then_serve(kernel):
    """A checkpoint's weights quantised, then prefill, decode through a
    captured graph and the grouped product on the same weights."""
    E, H, I, k = 8, 512, 256, 2
    g = gen(0)
    gate, up = (torch.randn((E, I, H), device=DEV, generator=g).mul_(H ** -0.5).to(BF) for _ in range(2))
    down = torch.randn((E, H, I), device=DEV, generator=g).mul_(I ** -0.5).to(BF)
    w13, w2, scales = mb.weights_from_checkpoint(list(gate), list(up), list(down), quantize="int4", group_size=64)
    assert w13.shape == (E, H // 2, 2 * I) and w2.shape == (E, I // 2, H) and w13.dtype == torch.uint8
    wide13 = mb.dequant_int4_groups(w13.transpose(1, 2).reshape(E * 2 * I, H // 2), scales[0].view(E * 2 * I, -1),
                                    dtype=torch.float32).double().view(E, 2 * I, H)
    # no weight is further from its 4-bit value than half a step, and the
    # scale's rounding moves seven steps by at most 7 u
    step = scales[0].double().repeat_interleave(64, dim=2)
    off = (wide13 - torch.cat((gate, up), dim=1).double()).abs()
    assert bool((off <= step * (0.5 + 7 * half_step(BF))).all())
    wide2 = mb.dequant_int4_groups(w2.transpose(1, 2).reshape(E * H, I // 2), scales[1].view(E * H, -1),
                                   dtype=torch.float32).double().view(E, H, I)
    for T in (1, 200):
        x = torch.randn((T, H), device=DEV, generator=gen(T)).to(BF)
        wts, ids = routing(T, E, k, T)
        ref, bound = layer_ref(x, wide13, wide2, wts, ids, BF)
        y = mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=scales)
        assert_within(y, ref, bound, BF)
        cap = mb.CapturedMoeMLP(w13, w2, T, k, scales=scales)
        assert torch.equal(cap(x, wts, ids), y)
        wts2, ids2 = routing(T, E, k, T + 1)
        x2 = x.flip(0) * 2
        assert torch.equal(cap(x2, wts2, ids2), mb.fused_moe_mlp(x2, w13, w2, wts2, ids2, scales=scales))


def test_two_captured_graphs_do_not_share_state(kernel):
    E, H, I, k = 8, 256, 128, 2
    w13, s13, _ = weights(E, 2 * I, H, 128, BF, 1)
    w2, s2, _ = weights(E, H, I, 128, BF, 2)
    caps, want, args = [], [], []
    for T in (4, 600):
        x = torch.randn((T, H), device=DEV, generator=gen(T)).to(BF)
        wts, ids = routing(T, E, k, T)
        caps.append(mb.CapturedMoeMLP(w13, w2, T, k, scales=(s13, s2)))
        want.append(mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2)))
        args.append((x, wts, ids))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, a, st in zip(caps, args, streams):
            with torch.cuda.stream(st):
                c(*a)
    torch.cuda.synchronize()
    assert torch.equal(caps[0].y, want[0]) and torch.equal(caps[1].y, want[1])


def test_calls_on_several_streams_at_once(kernel):
    E, H, I, k = 8, 512, 256, 2
    w13, s13, _ = weights(E, 2 * I, H, 128, BF, 1)
    w2, s2, _ = weights(E, H, I, 128, BF, 2)
    xs = [torch.randn((T, H), device=DEV, generator=gen(T)).to(BF) for T in (1, 16, 300)]
    rt = [routing(x.shape[0], E, k, 7) for x in xs]
    want = [mb.fused_moe_mlp(x, w13, w2, *r, scales=(s13, s2)) for x, r in zip(xs, rt)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for x, r, st in zip(xs, rt, streams):
            with torch.cuda.stream(st):
                got.append(mb.fused_moe_mlp(x, w13, w2, *r, scales=(s13, s2)))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 3])


def test_torch_op_takes_4_bit_weights(kernel):
    E, H, I, k, T = 4, 256, 128, 2, 6
    w13, s13, _ = weights(E, 2 * I, H, 128, BF, 1)
    w2, s2, _ = weights(E, H, I, 128, BF, 2)
    x = torch.randn((T, H), device=DEV, generator=gen(3)).to(BF)
    wts, ids = routing(T, E, k, 4)

    def step(x, wts, ids):
        return mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2)) + 1

    want = step(x, wts, ids)
    assert torch.equal(torch.compile(step, fullgraph=True, backend="aot_eager")(x, wts, ids), want)
    sizes = torch.tensor([1, 2, 0, 3], device=DEV)
    assert torch.equal(torch.ops.mail_b200.fused_moe_mlp_int4(x, w13, w2, sizes, s13, s2),
                       mb.fused_moe_mlp(x, w13, w2, sizes, scales=(s13, s2)))


def test_refusals_on_the_device():
    E, H, I, k, T = 4, 256, 128, 2, 6
    w13, s13, _ = weights(E, 2 * I, H, 128, BF, 1)
    w2, s2, _ = weights(E, H, I, 128, BF, 2)
    x = torch.randn((T, H), device=DEV, generator=gen(3)).to(BF)
    wts, ids = routing(T, E, k, 4)
    with pytest.raises(ValueError, match="scales"):
        mb.fused_moe_mlp(x, w13, w2, wts, ids)
    with pytest.raises(TypeError, match="share the activations' type"):
        mb.fused_moe_mlp(x.half(), w13, w2, wts, ids, scales=(s13, s2))
    with pytest.raises(TypeError, match="bf16 or fp16"):
        mb.fused_moe_mlp(x.float(), w13, w2, wts, ids, scales=(s13, s2))
    with pytest.raises(ValueError, match="group_size 256"):
        mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13[:, :, :1], s2[:, 1:]))
    with pytest.raises(ValueError, match="do not fit"):
        mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2[:, 1:]))
    with pytest.raises(ValueError, match="share a group size"):
        mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2.repeat_interleave(2, dim=2)))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        mb.grouped_matmul_int4(x, w13, s13, torch.tensor([1, 2, 0, 3], device=DEV).cpu().pin_memory())
    with pytest.raises(TypeError, match="unsupported dtype"):
        mb.fused_expert_rows(x, w13, w2, ids[:, 0], scales=(s13, s2))


def test_option_picks_the_kernel_and_its_default_stays():
    lib = _lib.load()
    assert lib.moe_get_option(_lib.OPT_INT4_GEMM) == 2
    assert lib.moe_set_option(_lib.OPT_INT4_GEMM, 3) == 1


@pytest.mark.parametrize("T,E,k", [(1, 4, 1), (32, 64, 1), (33, 64, 1), (32, 4, 4), (64, 128, 8), (130, 16, 8),
                                   (40, 300, 3), (2500, 8, 8)])
def test_layer_around_the_rules(T, E, k):
    """Sizes on both sides of the rules that choose a kernel: 32 tokens, 256
    and 1024 slots, eight rows an expert."""
    H, I, group = 256, 128, 64
    w13, s13, wide13 = weights(E, 2 * I, H, group, BF, 1)
    w2, s2, wide2 = weights(E, H, I, group, BF, 2)
    x = torch.randn((T, H), device=DEV, generator=gen(3)).to(BF)
    wts, ids = routing(T, E, k, 4)
    ref, bound = layer_ref(x, wide13, wide2, wts, ids, BF)
    assert_within(mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2)), ref, bound, BF)


def test_empty_batches():
    w13, s13, _ = weights(4, 256, 128, 64, BF, 1)
    w2, s2, _ = weights(4, 128, 128, 64, BF, 2)
    x = torch.empty((0, 128), dtype=BF, device=DEV)
    ids = torch.empty((0, 2), dtype=torch.int32, device=DEV)
    y = mb.fused_moe_mlp(x, w13, w2, torch.empty((0, 2), device=DEV), ids, scales=(s13, s2))
    assert y.shape == (0, 128) and y.dtype == BF
    assert mb.fused_moe_mlp(x, w13, w2, torch.zeros(4, dtype=torch.int64, device=DEV),
                            scales=(s13, s2)).shape == (0, 128)
    with pytest.raises(ValueError, match="need scales"):
        mb.fused_moe_mlp(x, w13, w2, torch.zeros(4, dtype=torch.int64, device=DEV))


def test_layer_takes_other_routing_types_and_strides():
    """int64 ids, bf16 weights, strided activations, ids and weights: what the
    layer takes with other weights, it takes here."""
    E, H, I, k, T = 8, 256, 128, 2, 40
    w13, s13, wide13 = weights(E, 2 * I, H, 64, BF, 1)
    w2, s2, wide2 = weights(E, H, I, 64, BF, 2)
    x = torch.randn((2 * T, 2 * H), device=DEV, generator=gen(3)).to(BF)[::2, H:]
    wts, ids = routing(T, E, k, 4)
    want = mb.fused_moe_mlp(x.contiguous(), w13, w2, wts, ids, scales=(s13, s2))
    many = torch.stack((ids.long(), ids.long() + 1), dim=2)[:, :, 0]
    assert torch.equal(mb.fused_moe_mlp(x, w13, w2, wts.t().contiguous().t(), many, scales=(s13, s2)), want)
    rounded = mb.fused_moe_mlp(x, w13, w2, wts.to(BF).float(), ids, scales=(s13, s2))
    assert torch.equal(mb.fused_moe_mlp(x, w13, w2, wts.to(BF), ids, scales=(s13, s2)), rounded)
    grown = torch.cat((s13, s13), dim=2)[:, :, :s13.shape[2]]
    assert not grown.is_contiguous()
    assert torch.equal(mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(grown, s2)), want)


def test_misaligned_activations_are_refused():
    w, s, _ = weights(2, 32, 128, 64, BF, 1)
    x = torch.zeros(4 * 128 + 1, dtype=BF, device=DEV)[1:].view(4, 128)
    with pytest.raises(mb.MoeError, match="aligned"):
        mb.grouped_matmul_int4(x, w, s, torch.tensor([2, 2], device=DEV))


@pytest.mark.parametrize("repeats", [False, True])
@pytest.mark.parametrize("T,E,k,H", [(32, 32, 8, 256), (32, 32, 8, 1024), (32, 32, 8, 2048), (32, 32, 8, 4096),
                                     (20, 8, 3, 1024), (32, 128, 8, 2048), (100, 128, 8, 256)])
def test_decode_batch_with_crowded_experts(T, E, k, H, repeats):
    """33 slots and more with several tiles of rows for one expert: every CTA has
    to cut the same tiles from the routing, call after call. (The hidden sizes
    give clusters of eight, four or two CTAs a strip, and one alone.)"""
    I, group = 768, 64
    w13, s13, wide13 = weights(E, 2 * I, H, group, BF, 1)
    w2, s2, wide2 = weights(E, H, I, group, BF, 2)
    x = torch.randn((T, H), device=DEV, generator=gen(3)).to(BF)
    score = torch.rand((T, E), device=DEV, generator=gen(4))
    for e, rows in enumerate((32, 17, 16, 9)[:k - 1]):  # tokens that name expert e
        score[:, e] += 10 * (torch.randperm(T, device=DEV, generator=gen(5 + e)) < rows) - 5
    top, ids = torch.topk(score, k, dim=1)
    wts, ids = torch.softmax(top % 1, dim=1).float(), ids.to(torch.int32)
    if repeats:  # the first two slots of every other token name one expert, some slots none
        ids[::2, 1] = ids[::2, 0]
        ids[1::4, -1] = -1
    assert 32 < T * k <= 8 * E
    ref, bound = layer_ref(x, wide13, wide2, wts, ids, BF)
    first = mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2))
    assert_within(first, ref, bound, BF)
    differ = torch.zeros((), dtype=torch.int64, device=DEV)
    for _ in range(400):
        differ += (mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2)) != first).any()
    assert int(differ) == 0, f"{int(differ)} of 400 calls differ from the first"
    assert mb.device_error() == 0


@pytest.mark.parametrize("T,group", [(2, 32), (9, 128), (30, 64)])
@pytest.mark.parametrize("power", [119, 124, 127])
def test_grouped_matmul_takes_activations_up_to_the_largest(power, T, group, kernel):
    """bf16 activations just below the type's largest: sums that fit come out,
    exactly (all terms are multiples of 2^(power - 14) and their sums below
    2^(power + 1), so fp32 holds them and no partial sum overflows)."""
    K, N = 384, 40
    w, s, wide = weights(2, N, K, group, BF, 3, exact=True)
    s, wide = s * 2.0 ** -12, wide * 2.0 ** -12
    x = (torch.randint(-1, 2, (T, K), device=DEV, generator=gen(T)).double() * 2.0 ** power).to(BF)
    ref, mag = grouped_ref(x, wide, [T - 1, 1])
    assert float(mag.max()) < 2.0 ** min(power + 1, 128)
    out = mb.grouped_matmul_int4(x, w, s, torch.tensor([T - 1, 1], device=DEV))
    assert torch.equal(out, ref.to(BF))


@pytest.mark.parametrize("T", [1, 20, 40])
def test_layer_takes_large_hidden_values(T, kernel):
    """Rows of h near 2^121 (bf16): the down projection's sums stay finite."""
    E, k, H, I, group = 16, 3, 256, 384, 128
    w13, s13, wide13 = weights(E, 2 * I, H, group, BF, 1)
    w2, s2, wide2 = weights(E, H, I, group, BF, 2)
    x = (torch.randn((T, H), device=DEV, generator=gen(3)) * 2.0 ** 60).to(BF)
    wts, ids = routing(T, E, k, 4)
    ref, bound = layer_ref(x, wide13, wide2, wts, ids, BF)
    assert 2.0 ** 118 < float(ref.abs().max()) < 2.0 ** 126
    assert_within(mb.fused_moe_mlp(x, w13, w2, wts, ids, scales=(s13, s2)), ref, bound, BF)


@pytest.mark.parametrize("power", [-100, -118, -126])
def test_grouped_matmul_takes_small_activations(power, kernel):
    """bf16 activations down to the smallest normal number. Terms are multiples
    of 2^(power - 2); what a sum may lose is half of bf16's smallest step."""
    T, K, N = 5, 256, 40
    w, s, wide = weights(2, N, K, 128, BF, 3, exact=True)
    x = (torch.randint(-2, 3, (T, K), device=DEV, generator=gen(T)).double() * 2.0 ** power).to(BF)
    ref, _ = grouped_ref(x, wide, [T - 1, 1])
    out = mb.grouped_matmul_int4(x, w, s, torch.tensor([T - 1, 1], device=DEV))
    assert_within(out, ref, torch.zeros_like(ref), BF)


def in_a_new_thread(call):
    import threading

    got = []

    def work():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001  (handed to the caller)
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.mark.parametrize("entry", ["C", "product", "layer", "bf16"])
def test_first_cuda_call_of_a_host_thread(entry, kernel):
    """A thread that has made no CUDA call yet calls the library first."""
    E, K, N, T = 2, 128, 256, 24
    w, s, wide = weights(E, N, K, 64, BF, 1, exact=True)
    w2, s2, _ = weights(E, K, N // 2, 64, BF, 2, exact=True)
    x = small_ints((T, K), BF, 3)
    gs = torch.tensor([20, 4], dtype=torch.int32, device=DEV)
    lib = _lib.load()
    if entry == "C":
        out = torch.zeros((T, N), dtype=BF, device=DEV)
        torch.cuda.synchronize()
        rc = in_a_new_thread(lambda: (lib.moe_grouped_matmul_int4(
            x.data_ptr(), _lib.BF16, T, K, w.data_ptr(), s.data_ptr(), 64, E, N, gs.data_ptr(), _lib.I32,
            out.data_ptr(), None), lib.moe_last_error().decode()))
        assert rc[0] == 0, rc[1]
        torch.cuda.synchronize()
        assert torch.equal(out, grouped_ref(x, wide, [20, 4])[0].to(BF))
        return
    if entry == "product":
        def call():
            return mb.grouped_matmul_int4(x, w, s, gs)
    elif entry == "layer":
        def call():
            return mb.fused_moe_mlp(x, w, w2, gs, scales=(s, s2))
    else:
        a, b = wide.to(BF).transpose(1, 2), torch.zeros((E, K, N // 2), dtype=BF, device=DEV).transpose(1, 2)

        def call():
            return mb.fused_moe_mlp(x, a, b, gs)
    torch.cuda.synchronize()
    assert torch.equal(in_a_new_thread(call), call())


def test_tiles_of_different_sizes_from_two_host_threads():
    """The shared memory of a launch depends on the number of experts; threads
    whose layers differ do not get in each other's way."""
    import threading

    lib = _lib.load()
    before = lib.moe_get_option(_lib.OPT_INT4_GEMM)
    assert lib.moe_set_option(_lib.OPT_INT4_GEMM, 1) == 0
    K, N, T, jobs, streams = 128, 64, 64, [], []
    for E in (2, 512):
        w, s, wide = weights(E, N, K, 128, BF, E, exact=True)
        x = small_ints((T, K), BF, E)
        gs = torch.tensor([0] * (E - 1) + [T], dtype=torch.int32, device=DEV)
        out = torch.empty((T, N), dtype=BF, device=DEV)
        streams.append(torch.cuda.Stream())
        args = (x.data_ptr(), _lib.BF16, T, K, w.data_ptr(), s.data_ptr(), 128, E, N, gs.data_ptr(), _lib.I32,
                out.data_ptr(), streams[-1].cuda_stream)
        jobs.append((args, out, (x.double() @ wide[-1].t()).to(BF), (w, s, x, gs)))
    torch.cuda.synchronize()
    failed = []

    def work(args):
        for _ in range(20000):
            if lib.moe_grouped_matmul_int4(*args) != 0:
                failed.append(lib.moe_last_error().decode())
                return

    threads = [threading.Thread(target=work, args=(j[0],)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert lib.moe_set_option(_lib.OPT_INT4_GEMM, before) == 0
    assert not failed, failed[0]
    for _, out, ref, _ in jobs:
        assert torch.equal(out, ref)
    assert mb.device_error() == 0


def full_scales(shape, bits, dtype, seed):
    """Scales with all `bits` significant bits in one binade: multiples of
    2^(1 - bits) in [1, 2)."""
    m = torch.randint(2 ** (bits - 1), 2 ** bits, shape, device=DEV, generator=gen(seed))
    return (m.double() * 2.0 ** (1 - bits)).to(dtype)


@pytest.fixture
def row_kernels():
    lib = _lib.load()
    before = lib.moe_get_option(_lib.OPT_INT4_GEMM)
    assert lib.moe_set_option(_lib.OPT_INT4_GEMM, 0) == 0
    yield
    assert mb.device_error() == 0
    assert lib.moe_set_option(_lib.OPT_INT4_GEMM, before) == 0


@pytest.mark.parametrize("dtype,bits", [(BF, 8), (HF, 11)])
@pytest.mark.parametrize("K,N,group,sizes", [(32, 70, 32, [3]), (384, 40, 128, [1, 0, 2]), (384, 33, 64, [9, 17]),
                                             (512, 50, 32, [40, 1])])
def test_row_kernels_round_no_weight(dtype, bits, K, N, group, sizes, row_kernels):
    """Scales with a full significand: (q - 8) s needs more bits than the
    activations' type has. All terms are multiples of 2^(1 - bits), and the sums
    of their magnitudes below 2^24 of these, so fp32 holds every sum: the output
    has to be the exact result, rounded once."""
    E, T = len(sizes), sum(sizes)
    w, _, wide = weights(E, N, K, group, dtype, K + N, exact=False)
    q = torch.stack((w.transpose(1, 2) & 15, w.transpose(1, 2) >> 4), dim=-1).view(E, N, K)
    s = full_scales((E, N, K // group), bits, dtype, N)
    wide = (q.double() - 8) * s.double().repeat_interleave(group, dim=2)
    assert bool((wide.to(dtype).double() != wide).any())
    x = small_ints((T, K), dtype, T)
    ref, mag = grouped_ref(x, wide, sizes)
    assert float(mag.max()) * 2 ** (bits - 1) < 2 ** 24
    out = mb.grouped_matmul_int4(x, w, s, torch.tensor(sizes, dtype=torch.int32, device=DEV))
    assert torch.equal(out, ref.to(dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,E,k", [(1, 4, 1), (3, 4, 4), (20, 8, 4), (32, 32, 8), (40, 6, 3)])
def test_decode_layer_rounds_no_weight(dtype, T, E, k, row_kernels):
    """A layer whose h is exact (gates are 128, where silu(g) = g; h = 128 u with
    |u| <= 32 whole) and whose down weights need more bits than the type has. The
    terms are multiples of 2^-3, all sums below 2^21."""
    H, I, group = 64, 64, 32
    g = gen(T)
    q13 = torch.randint(0, 16, (E, 2 * I, H), device=DEV, generator=g)
    q13[:, :I] = 8
    q13[:, :I, 0] = 12   # gate = 4 * 2 * x[0]
    q13[:, I:, 0] = 8
    s13 = torch.ones((E, 2 * I, H // group), device=DEV)
    s13[:, :I] = 2
    w13 = (q13[..., 0::2] | (q13[..., 1::2] << 4)).to(torch.uint8).transpose(1, 2)
    w2, _, _ = weights(E, H, I, group, dtype, 2)
    q2 = torch.stack((w2.transpose(1, 2) & 15, w2.transpose(1, 2) >> 4), dim=-1).view(E, H, I)
    s2 = full_scales((E, H, I // group), 8, dtype, 3)
    wide2 = (q2.double() - 8) * s2.double().repeat_interleave(group, dim=2)
    x = torch.zeros((T, H), device=DEV)
    x[:, 1:5] = torch.randint(-1, 2, (T, 4), device=DEV, generator=g).float()
    x[:, 0] = 16
    _, ids = routing(T, E, k, 4)
    wts = torch.tensor([0.5, 0.25, 0.125], device=DEV)[torch.randint(0, 3, (T, k), device=DEV, generator=g)]
    ref = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(ref)
    for j in range(k):
        u = torch.einsum("th,tnh->tn", x.double(), q13[ids[:, j].long(), I:].double() - 8)
        assert float(u.abs().max()) <= 32
        o = torch.einsum("ti,tni->tn", 128 * u, wide2[ids[:, j].long()])
        m = torch.einsum("ti,tni->tn", 128 * u.abs(), wide2[ids[:, j].long()].abs())
        ref += wts[:, j:j + 1].double() * o
        mag += wts[:, j:j + 1].double() * m
    assert float(mag.max()) * 2 ** 3 < 2 ** 24
    y = mb.fused_moe_mlp(x.to(dtype), w13, w2, wts, ids, scales=(s13.to(dtype), s2))
    assert torch.equal(y, ref.to(dtype))


def test_grouped_matmul_spreads_an_infinity_over_its_row_only(kernel):
    """q = 8 makes 0 * inf = NaN of it, every other weight an infinity; rows of
    the same tile keep their values."""
    w, s, wide = weights(2, 64, 256, 128, BF, 5, exact=True)
    x = small_ints((20, 256), BF, 3)
    ref, _ = grouped_ref(x, wide, [9, 11])
    for r, c, v in ((2, 0, float("inf")), (15, 200, float("inf")), (19, 255, -float("inf"))):
        x[r, c] = v
    out = mb.grouped_matmul_int4(x, w, s, torch.tensor([9, 11], device=DEV))
    rows = [r for r in range(20) if r not in (2, 15, 19)]
    assert torch.equal(out[rows], ref.to(BF)[rows])
    assert not bool(torch.isfinite(out[[2, 15, 19]]).any())


def test_grouped_matmul_takes_fp16_scales_up_to_8188(kernel):
    """-8 * 8188 is fp16's largest number: up to there the tiles hold every
    weight, and exactly where the step is a power of two."""
    K, N, T = 64, 40, 12
    q = torch.tensor([0, 4, 6, 7, 8, 9, 10, 12], device=DEV)[torch.randint(0, 8, (N, K), device=DEV, generator=gen(5))]
    s = torch.full((1, N, K // 32), 8188.0, dtype=HF, device=DEV)
    w = (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8).view(1, N, K // 2).transpose(1, 2)
    wide = (q.double() - 8) * 8188
    assert torch.equal(wide.to(HF).double(), wide) and float(wide.min()) == -65504
    x = (small_ints((T, K), HF, 3).double() * 2.0 ** -8).to(HF)
    ref = x.double() @ wide.t()
    assert torch.equal(mb.grouped_matmul_int4(x, w, s, torch.tensor([T], device=DEV)), ref.to(HF))
