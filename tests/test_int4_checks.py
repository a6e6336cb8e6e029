"""4-bit expert weights: what the entry points refuse, checked on the host
without a GPU, and the shapes of the registered operators."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import mail_b200 as mb  # noqa: E402
from mail_b200 import _lib, int4  # noqa: E402

P = ctypes.c_void_p(16)
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("call,needle", [
    (lambda L: L.moe_quant_int4_groups(P, _lib.I8, 4, 128, 128, P, P, _lib.BF16, None), "source must be"),
    (lambda L: L.moe_quant_int4_groups(P, _lib.BF16, 4, 128, 128, P, P, _lib.F32, None), "scales must be"),
    (lambda L: L.moe_quant_int4_groups(P, _lib.BF16, 4, 128, 16, P, P, _lib.BF16, None), "group size 16"),
    (lambda L: L.moe_quant_int4_groups(P, _lib.BF16, 4, 96, 64, P, P, _lib.BF16, None), "multiple of the group"),
    (lambda L: L.moe_quant_int4_groups(None, _lib.BF16, 4, 128, 64, P, P, _lib.BF16, None), "NULL"),
    (lambda L: L.moe_quant_int4_groups(ctypes.c_void_p(8), _lib.BF16, 4, 128, 64, P, P, _lib.BF16, None), "aligned"),
    (lambda L: L.moe_dequant_int4_groups(P, P, _lib.BF16, 4, 128, 64, P, _lib.I8, None), "output must be"),
    (lambda L: L.moe_dequant_int4_groups(P, P, _lib.F32, 4, 128, 64, P, _lib.F32, None), "scales must be"),
    (lambda L: L.moe_dequant_int4_groups(P, None, _lib.BF16, 4, 128, 64, P, _lib.F32, None), "NULL"),
    (lambda L: L.moe_grouped_matmul_int4(P, _lib.F32, 4, 128, P, P, 128, 2, 8, P, _lib.I32, P, None), "bf16 or fp16"),
    (lambda L: L.moe_grouped_matmul_int4(P, _lib.BF16, 4, 100, P, P, 32, 2, 8, P, _lib.I32, P, None), "multiple"),
    (lambda L: L.moe_grouped_matmul_int4(P, _lib.BF16, 4, 128, P, P, 128, 0, 8, P, _lib.I32, P, None), "num_experts"),
    (lambda L: L.moe_grouped_matmul_int4(P, _lib.BF16, 4, 128, P, P, 128, 1025, 8, P, _lib.I32, P, None),
     "num_experts"),
    (lambda L: L.moe_grouped_matmul_int4(P, _lib.BF16, 4, 128, P, P, 128, 2, 0, P, _lib.I32, P, None), "output size"),
    (lambda L: L.moe_grouped_matmul_int4(P, _lib.BF16, 4, 128, P, P, 128, 2, 8, P, _lib.F32, P, None), "group sizes"),
    (lambda L: L.moe_grouped_matmul_int4(P, _lib.BF16, 4, 128, None, P, 128, 2, 8, P, _lib.I32, P, None), "NULL"),
    (lambda L: L.moe_grouped_matmul_int4(P, _lib.BF16, 4, 128, ctypes.c_void_p(8), P, 128, 2, 8, P, _lib.I32, P,
                                         None), "aligned"),
    (lambda L: L.moe_fused_experts_int4(P, _lib.BF16, 4, 128, P, P, P, P, 128, 2, 96, P, P, 2, P, P, 1 << 30, None),
     "multiple"),
    (lambda L: L.moe_fused_experts_int4(P, _lib.BF16, 4, 128, P, P, P, P, 128, 2, 128, P, P, 0, P, P, 1 << 30, None),
     "bad sizes"),
    (lambda L: L.moe_fused_experts_int4(P, _lib.BF16, 4, 128, P, P, P, P, 128, 2, 128, P, None, 2, P, P, 1 << 30,
                                        None), "NULL"),
    (lambda L: L.moe_fused_mlp_int4(P, _lib.BF16, 4, 128, P, P, P, P, 128, 2, 128, P, _lib.F16, P, P, 1 << 30, None),
     "group sizes"),
])
def test_invalid_arguments_are_rejected_on_host(call, needle):
    lib = _lib.load()
    assert call(lib) == 1  # MOE_ERR_INVALID_ARG
    assert needle in lib.moe_last_error().decode()


def test_small_workspace_is_refused():
    lib = _lib.load()
    need = lib.moe_fused_experts_int4_workspace_size(4, 128, 128, 2, 2)
    assert need > 0
    assert lib.moe_fused_experts_int4(P, _lib.BF16, 4, 128, P, P, P, P, 128, 2, 128, P, P, 2, P, P, need - 1, None) == 4
    need = lib.moe_fused_mlp_int4_workspace_size(4, 128, 2)
    assert lib.moe_fused_mlp_int4(P, _lib.BF16, 4, 128, P, P, P, P, 128, 2, 128, P, _lib.I32, P, P, need - 1, None) == 4
    assert lib.moe_fused_experts_int4_workspace_size(-1, 128, 128, 2, 2) == 0


def test_empty_batches_launch_nothing():
    lib = _lib.load()
    before = lib.moe_launch_count()
    assert lib.moe_quant_int4_groups(None, _lib.BF16, 0, 128, 64, None, None, _lib.BF16, None) == 0
    assert lib.moe_dequant_int4_groups(None, None, _lib.BF16, 0, 128, 64, None, _lib.F32, None) == 0
    assert lib.moe_grouped_matmul_int4(None, _lib.BF16, 0, 128, None, None, 128, 2, 8, None, _lib.I32, None, None) == 0
    assert lib.moe_fused_experts_int4(None, _lib.BF16, 0, 128, None, None, None, None, 128, 2, 128, None, None, 2,
                                      None, None, 0, None) == 0
    assert lib.moe_fused_mlp_int4(None, _lib.BF16, 0, 128, None, None, None, None, 128, 2, 128, None, _lib.I32, None,
                                  None, 0, None) == 0
    assert lib.moe_launch_count() == before


def test_cpu_tensors_are_refused():
    w = torch.zeros((4, 128), dtype=BF)
    q, s = torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 1), dtype=BF)
    with pytest.raises(ValueError, match="CUDA"):
        mb.quant_int4_groups(w)
    with pytest.raises(ValueError, match="CUDA"):
        mb.dequant_int4_groups(q, s)
    with pytest.raises(ValueError, match="CUDA"):
        mb.grouped_matmul_int4(w, q.view(1, 64, 4), s.view(1, 4, 1), torch.tensor([4]))
    with pytest.raises(ValueError, match="CUDA"):
        mb.fused_moe_mlp(w, torch.zeros((1, 64, 256), dtype=torch.uint8), torch.zeros((1, 64, 128), dtype=torch.uint8),
                         torch.tensor([4]), scales=(s, s))


@pytest.mark.parametrize("dtype,w,scale,K,err,needle", [
    (torch.float32, (2, 64, 8), (2, 8, 1), 128, TypeError, "bf16 or fp16"),
    (BF, (2, 32, 8), (2, 8, 1), 128, ValueError, "K = 128"),
    (BF, (2, 64), (2, 8, 1), 128, ValueError, "uint8"),
    (BF, (2, 64, 8), (2, 8), 128, ValueError, "do not fit"),
    (BF, (2, 64, 8), (2, 9, 1), 128, ValueError, "do not fit"),
    (BF, (2, 64, 8), (2, 8, 3), 128, ValueError, "do not fit"),
    (BF, (2, 64, 8), (2, 8, 0), 128, ValueError, "do not fit"),
    (BF, (2, 64, 8), (2, 8, 8), 128, ValueError, "group_size 16"),
])
def test_weight_and_scale_shapes(dtype, w, scale, K, err, needle):
    with pytest.raises(err, match=needle):
        int4._check_weight("op", dtype, torch.zeros(w, dtype=torch.uint8), torch.zeros(scale, dtype=dtype), K)


def test_scales_share_the_activations_type():
    w = torch.zeros((2, 64, 8), dtype=torch.uint8)
    with pytest.raises(TypeError, match="share"):
        int4._check_weight("op", BF, w, torch.zeros((2, 8, 1), dtype=HF), 128)
    assert int4._check_weight("op", HF, w, torch.zeros((2, 8, 4), dtype=HF), 128) == 32


def test_fake_kernels_know_4_bit_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty((6, 256), dtype=BF)
        w13 = torch.empty((4, 256, 128), dtype=torch.uint8).transpose(1, 2)  # [E, 2I, H / 2] bytes
        w2 = torch.empty((4, 256, 64), dtype=torch.uint8).transpose(1, 2)
        s13, s2 = torch.empty((4, 256, 2), dtype=BF), torch.empty((4, 256, 1), dtype=BF)
        ids = torch.empty((6, 2), dtype=torch.int32)
        y = torch.ops.mail_b200.fused_experts(x, w13, w2, torch.empty((6, 2)), ids, s13, s2)
        assert tuple(y.shape) == (6, 256) and y.dtype == BF
        y = torch.ops.mail_b200.fused_moe_mlp_int4(x, w13, w2, torch.empty(4, dtype=torch.int64), s13, s2)
        assert tuple(y.shape) == (6, 256)
        y = torch.ops.mail_b200.grouped_matmul_int4(x, w13, s13, torch.empty(4, dtype=torch.int64))
        assert tuple(y.shape) == (6, 256) and y.dtype == BF
        y, wts, i = torch.ops.mail_b200.fused_experts_from_logits(x, w13, w2, torch.empty((6, 4)), 2, "softmax", True,
                                                                  s13, s2)
        assert tuple(y.shape) == (6, 256) and tuple(wts.shape) == (6, 2) and i.dtype == torch.int32
        with pytest.raises(ValueError, match="shape mismatch"):
            torch.ops.mail_b200.fused_experts(x[:, :128], w13, w2, torch.empty((6, 2)), ids, s13, s2)


def test_checkpoint_quantize_argument():
    z = torch.zeros((1, 64, 64), dtype=BF)
    with pytest.raises(ValueError, match="quantize"):
        mb.weights_from_checkpoint(z, z, z, quantize="int3")
    with pytest.raises(ValueError, match="CUDA"):
        mb.weights_from_checkpoint(z, z, z, quantize="int4", group_size=64)


@pytest.mark.parametrize("quantize", [None, 0, "", [], 2, (1,), "int8"])
def test_checkpoint_quantize_is_taken_by_its_truth(quantize):
    """Any value that is no string is taken by its truth, as before there were
    names for the types; what asks for int8 gets as far as needing the device."""
    z = torch.zeros((1, 64, 64), dtype=BF)
    if quantize:
        with pytest.raises(ValueError, match="CUDA"):
            mb.weights_from_checkpoint(z, z, z, quantize=quantize)
    else:
        w13, w2 = mb.weights_from_checkpoint(z, z, z, quantize=quantize)
        assert w13.shape == (1, 64, 128) and w2.shape == (1, 64, 64) and w13.dtype == BF


def test_checkpoint_names_that_mean_nothing_are_refused():
    z = torch.zeros((1, 64, 64), dtype=BF)
    for name in ("int2", "fp8", "INT4"):
        with pytest.raises(ValueError, match="quantize"):
            mb.weights_from_checkpoint(z, z, z, quantize=name)


@pytest.mark.parametrize("scales", [(), (None,), (None, None, None), torch.zeros(3)])
def test_pre_routed_call_with_dense_weights_does_not_read_scales(scales):
    x, w13, w2 = (torch.zeros(s, dtype=BF) for s in ((4, 64), (2, 64, 128), (2, 64, 64)))
    with pytest.raises(ValueError, match="CUDA tensors only"):  # past the argument
        mb.fused_moe_mlp(x, w13, w2, torch.tensor([2, 2]), scales=scales)


def _fake(*shapes):
    return [torch.empty(s, dtype=d) for s, d in shapes]


@pytest.mark.parametrize("change,err,needle", [
    (dict(x=((256,), BF)), ValueError, "x \\[T, K\\]"),
    (dict(x=((2, 6, 256), BF)), ValueError, "x \\[T, K\\]"),
    (dict(gs=((3,), torch.int64)), ValueError, "E entries"),
    (dict(gs=((0,), torch.int64)), ValueError, "E entries"),
    (dict(w=((4, 64, 256), torch.uint8)), ValueError, "K = 256"),
    (dict(s=((4, 256, 2), HF)), TypeError, "share"),
])
def test_registered_product_refuses_when_traced(change, err, needle):
    from torch._subclasses.fake_tensor import FakeTensorMode

    args = dict(x=((6, 256), BF), w=((4, 128, 256), torch.uint8), s=((4, 256, 2), BF), gs=((4,), torch.int64))
    with FakeTensorMode():
        assert tuple(torch.ops.mail_b200.grouped_matmul_int4(*_fake(*args.values())).shape) == (6, 256)
        with pytest.raises(err, match=needle):
            torch.ops.mail_b200.grouped_matmul_int4(*_fake(*{**args, **change}.values()))


@pytest.mark.parametrize("change,err,needle", [
    (dict(x=((6, 256), torch.float32)), TypeError, "bf16 or fp16"),
    (dict(w2=((4, 64, 256), BF)), TypeError, "both be 4-bit"),
    (dict(s13=((4, 256, 3), BF)), ValueError, "do not fit"),
    (dict(s13=((4, 256, 2), HF)), TypeError, "share"),
    (dict(s2=((4, 128, 1), BF)), ValueError, "do not fit"),
    (dict(s2=((4, 256, 2), BF)), ValueError, "share a group size"),
    (dict(s2=None), ValueError, "need scales"),
])
@pytest.mark.parametrize("form", ["top-k", "logits", "pre-routed"])
def test_registered_layers_refuse_when_traced(form, change, err, needle):
    from torch._subclasses.fake_tensor import FakeTensorMode

    args = dict(x=((6, 256), BF), w13=((4, 128, 256), torch.uint8), w2=((4, 64, 256), torch.uint8),
                s13=((4, 256, 2), BF), s2=((4, 256, 1), BF))
    ops = torch.ops.mail_b200

    def call(a):
        x, w13, w2, s13, s2 = (None if v is None else torch.empty(v[0], dtype=v[1]) for v in a.values())
        if form == "top-k":
            return ops.fused_experts(x, w13, w2, torch.empty((6, 2)), torch.empty((6, 2), dtype=torch.int32), s13, s2)
        if form == "logits":
            return ops.fused_experts_from_logits(x, w13, w2, torch.empty((6, 4)), 2, "softmax", True, s13, s2)[0]
        return ops.fused_moe_mlp_int4(x, w13, w2, torch.empty(4, dtype=torch.int64), s13, s2)

    if form == "pre-routed" and change.get("s2", 0) is None:
        return  # that operator's scales are not optional
    with FakeTensorMode():
        assert tuple(call(args).shape) == (6, 256)
        with pytest.raises(err, match=needle):
            call({**args, **change})
