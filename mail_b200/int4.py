"""Experts with 4-bit weights and group scales (w4a16).

A weight row of K values is stored as K / 2 bytes and K / group_size scales:

    W[n, k] = (q[n, k] - 8) * scale[n, k // group_size],   q in 0..15

byte b of the row holds q[2b] in its low and q[2b + 1] in its high nibble;
group_size is 32, 64 or 128 and divides K; the scales are in the activations'
type (bf16 or fp16). Expert weights keep the framework's "(E, K, N)" logical
layout with K-major storage, so a 4-bit w13 is a uint8 [E, H / 2, 2I] view of
contiguous [E, 2I, H / 2] bytes with scales [E, 2I, H / group_size], and w2 is
[E, I / 2, H] with scales [E, H, I / group_size]. `fused_moe_mlp` and
`fused_moe_mlp_from_logits` take such weights with scales=(w13_scale, w2_scale).

Up to eight rows an expert on average are multiplied without rounding a weight;
with more, each weight is rounded once to the activations' type (in fp16 one
beyond 65504, from a scale above 8188, is infinite there).

Every op runs the kernels of libmoe_b200.so on the current stream of its
tensors' device; there is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import torch

from . import _lib
from .moe import _check_shapes, _require_cuda, _stream, kmajor

GROUP_SIZES = (32, 64, 128)
_ACT = (torch.bfloat16, torch.float16)
_CODES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _launch(dev: torch.device, name: str, *args) -> None:
    """The C call with `args` and the current stream of `dev`, with `dev` current.
    (A decode step is a few microseconds of kernels, so the host's share of a
    call counts: the stream is read as an integer, without a Stream object.)"""
    if dev.index == torch.cuda.current_device():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, _stream(dev))


def _one_device(name: str, *ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    for t in ts:
        if not t.is_cuda:
            _require_cuda(t)
        if t.device != dev:
            raise ValueError(f"{name}: all tensors must be on one device")
    return dev


def _kmajor(w: torch.Tensor) -> torch.Tensor:
    """w itself where its storage is K-major (the same first byte as the [E, N, K / 2]
    view's), a K-major copy otherwise."""
    E, K2, N = w.shape
    s0, s1, s2 = w.stride()
    return w if s1 == 1 and s2 == K2 and (s0 == K2 * N or E == 1) else kmajor(w)


def _check_group(name: str, K: int, group_size: int) -> None:
    if group_size not in GROUP_SIZES:
        raise ValueError(f"{name}: group_size {group_size} is not one of {GROUP_SIZES}")
    if K <= 0 or K % group_size:
        raise ValueError(f"{name}: the reduction length {K} must be a positive multiple of group_size {group_size}")


def quant_int4_groups(w: torch.Tensor, group_size: int = 128, scale_dtype: torch.dtype | None = None):
    """Rows [R, C] (bf16, fp16 or fp32) -> (q uint8 [R, C / 2], scale [R, C / group_size]).

    scale = absmax / 7 of each group (fp32 quotient, rounded to scale_dtype:
    w's type, or bf16 for fp32 weights), q = 8 + clamp(w / scale rounded half
    to even, -8, 7), 8 where the scale is 0. A group that holds a NaN or an
    infinity, or whose scale scale_dtype cannot hold, gets a NaN scale."""
    _require_cuda(w)
    if w.dim() != 2 or w.dtype not in (*_ACT, torch.float32):
        raise ValueError("quant_int4_groups: expected bf16, fp16 or fp32 weights [R, C]")
    scale_dtype = scale_dtype or (w.dtype if w.dtype in _ACT else torch.bfloat16)
    if scale_dtype not in _ACT:
        raise TypeError(f"quant_int4_groups: scales must be bf16 or fp16, not {scale_dtype}")
    R, C = w.shape
    _check_group("quant_int4_groups", C, group_size)
    w = w.contiguous()
    q = torch.empty((R, C // 2), dtype=torch.uint8, device=w.device)
    s = torch.empty((R, C // group_size), dtype=scale_dtype, device=w.device)
    _launch(w.device, "moe_quant_int4_groups", w.data_ptr(), _CODES[w.dtype], R, C, group_size, q.data_ptr(),
            s.data_ptr(), _CODES[scale_dtype])
    return q, s


def dequant_int4_groups(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """(q uint8 [R, C / 2], scale [R, C / group_size]) -> the values [R, C] they
    stand for, in dtype (the scales' type by default; each product is rounded
    to it once)."""
    dev = _one_device("dequant_int4_groups", q, scale)
    if q.dim() != 2 or q.dtype != torch.uint8 or scale.dim() != 2 or scale.dtype not in _ACT:
        raise ValueError("dequant_int4_groups: expected q uint8 [R, C / 2] and bf16 or fp16 scales [R, C / group_size]")
    R, C = q.shape[0], 2 * q.shape[1]
    if scale.shape[0] != R or scale.shape[1] == 0 or C % scale.shape[1]:
        raise ValueError(f"dequant_int4_groups: scales {tuple(scale.shape)} do not fit q {tuple(q.shape)}")
    group_size = C // scale.shape[1]
    _check_group("dequant_int4_groups", C, group_size)
    out = torch.empty((R, C), dtype=dtype or scale.dtype, device=dev)
    if out.dtype not in (*_ACT, torch.float32):
        raise TypeError(f"dequant_int4_groups: dtype must be bf16, fp16 or fp32, not {out.dtype}")
    q, scale = q.contiguous(), scale.contiguous()
    _launch(dev, "moe_dequant_int4_groups", q.data_ptr(), scale.data_ptr(), _CODES[scale.dtype], R, C, group_size,
            out.data_ptr(), _CODES[out.dtype])
    return out


def quantize_weights_int4(w13: torch.Tensor, w2: torch.Tensor, group_size: int = 128,
                          scale_dtype: torch.dtype | None = None):
    """Load-time weight prep: logical (E, K, N) weights -> 4-bit logical views
    with K-major storage and their group scales (quant_int4_groups on the
    K-major rows). Returns (w13_q [E, H / 2, 2I], w2_q [E, I / 2, H],
    (w13_scale [E, 2I, H / group_size], w2_scale [E, H, I / group_size]))."""
    def pack(w):
        wk = kmajor(w)
        E, N, K = wk.shape
        q, s = quant_int4_groups(wk.reshape(E * N, K), group_size, scale_dtype)
        return q.view(E, N, K // 2).transpose(1, 2), s.view(E, N, K // group_size)
    a, sa = pack(w13)
    b, sb = pack(w2)
    return a, b, (sa, sb)


def _check_weight(name: str, dtype: torch.dtype, w: torch.Tensor, scale: torch.Tensor, K: int) -> int:
    """Group size of a 4-bit weight [E, K / 2, N] with scales [E, N, K / g]."""
    if dtype not in _ACT:
        raise TypeError(f"{name}: 4-bit weights take bf16 or fp16 activations, not {dtype}")
    ws, ss = w.shape, scale.shape
    if len(ws) != 3 or w.dtype != torch.uint8 or 2 * ws[1] != K:
        raise ValueError(f"{name}: expected 4-bit weights uint8 [E, K / 2, N] with K = {K}, "
                         f"got {w.dtype} {tuple(ws)}")
    if scale.dtype != dtype:
        raise TypeError(f"{name}: the scales must share the activations' type {dtype}, not {scale.dtype}")
    if len(ss) != 3 or ss[0] != ws[0] or ss[1] != ws[2] or ss[2] == 0 or K % ss[2]:
        raise ValueError(f"{name}: scales {tuple(ss)} do not fit weights {tuple(ws)} "
                         "(expected [E, N, K / group_size])")
    group_size = K // ss[2]
    _check_group(name, K, group_size)
    return group_size


def _check_counts(name: str, group_sizes: torch.Tensor, E: int) -> None:
    if group_sizes.numel() != E:
        raise ValueError(f"{name}: group_sizes must have E entries")


def _counts(group_sizes: torch.Tensor) -> torch.Tensor:
    if group_sizes.dtype not in (torch.int32, torch.int64):
        group_sizes = group_sizes.to(torch.int64)
    return group_sizes.contiguous()


def grouped_matmul_int4(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor,
                        group_sizes: torch.Tensor) -> torch.Tensor:
    """Matrix product grouped by expert, with 4-bit weights: x [T, K] (bf16 or
    fp16) holds the rows of expert 0, then those of expert 1, and so on;
    group_sizes [E] says how many each has (any number, zero included; counts
    past T are cut off). Returns [T, N] in x's type,

        out[r, n] = sum_k x[r, k] * W[e(r), k, n]

    with w uint8 [E, K / 2, N] (K-major storage) and scale [E, N, K / group_size];
    rows behind the last group are zero. Under torch.compile the call is one
    operator (torch.ops.mail_b200.grouped_matmul_int4)."""
    if torch.compiler.is_compiling():
        return torch.ops.mail_b200.grouped_matmul_int4(x, w, scale, group_sizes)
    return _grouped_impl(x, w, scale, group_sizes)


def _check_grouped(x, w, scale, group_sizes) -> int:
    """Group size of a grouped product's weights, its arguments checked."""
    name = "grouped_matmul_int4"
    if x.dim() != 2:
        raise ValueError(f"{name}: expected x [T, K]")
    group_size = _check_weight(name, x.dtype, w, scale, x.shape[1])
    _check_counts(name, group_sizes, w.shape[0])
    return group_size


def _grouped_impl(x, w, scale, group_sizes):
    dev = _one_device("grouped_matmul_int4", x, w, scale, group_sizes)
    group_size = _check_grouped(x, w, scale, group_sizes)
    T, K = x.shape
    E, _, N = w.shape
    gs = _counts(group_sizes)
    x, wk, scale = x.contiguous(), _kmajor(w), scale.contiguous()
    out = torch.empty((T, N), dtype=x.dtype, device=dev)
    _launch(dev, "moe_grouped_matmul_int4", x.data_ptr(), _CODES[x.dtype], T, K, wk.data_ptr(), scale.data_ptr(),
            group_size, E, N, gs.data_ptr(), _lib.I32 if gs.dtype == torch.int32 else _lib.I64, out.data_ptr())
    return out


def check_layer(x, w13, w2, w13_scale, w2_scale) -> int:
    """Group size of a layer's 4-bit weights, types and scales checked (the
    shapes of x, w13 and w2 by _check_shapes)."""
    name = "fused_moe_mlp"
    if w13_scale is None or w2_scale is None:
        raise ValueError(f"{name}: 4-bit weights need scales=(w13_scale, w2_scale)")
    if w2.dtype != torch.uint8:
        raise TypeError(f"{name}: w13 and w2 must both be 4-bit (uint8)")
    group = _check_weight(name, x.dtype, w13, w13_scale, x.shape[1])
    if _check_weight(name, x.dtype, w2, w2_scale, w13.shape[2] // 2) != group:
        raise ValueError(f"{name}: w13 and w2 must share a group size")
    return group


def _layer_weights(x, w13, w2, w13_scale, w2_scale):
    """(E, H, I, group size, K-major w13, scales, K-major w2, scales), checked."""
    group = check_layer(x, w13, w2, w13_scale, w2_scale)
    E, _, two_i = w13.shape
    return E, x.shape[1], two_i // 2, group, _kmajor(w13), w13_scale.contiguous(), _kmajor(w2), w2_scale.contiguous()


def fused_experts(x, w13, w2, topk_weights, topk_ids, w13_scale, w2_scale):
    """The top-k form of fused_moe_mlp with 4-bit weights (shapes checked by
    the caller)."""
    E, H, inter, group, a, sa, b, sb = _layer_weights(x, w13, w2, w13_scale, w2_scale)
    dev = _one_device("fused_moe_mlp", x, w13, w2, topk_weights, topk_ids, w13_scale, w2_scale)
    x = x.contiguous()
    wts = topk_weights if topk_weights.dtype == torch.float32 else topk_weights.to(torch.float32)
    ids = topk_ids if topk_ids.dtype == torch.int32 else topk_ids.to(torch.int32)
    wts, ids = wts.contiguous(), ids.contiguous()
    T, k = ids.shape
    y = x.new_empty((T, H))
    size = _lib.query("moe_fused_experts_int4_workspace_size", T, H, inter, E, k)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _launch(dev, "moe_fused_experts_int4", x.data_ptr(), _CODES[x.dtype], T, H, a.data_ptr(), sa.data_ptr(),
            b.data_ptr(), sb.data_ptr(), group, E, inter, wts.data_ptr(), ids.data_ptr(), k, y.data_ptr(),
            ws.data_ptr(), size)
    return y


def fused_mlp(x, w13, w2, group_sizes, w13_scale, w2_scale):
    """The pre-routed form of fused_moe_mlp with 4-bit weights."""
    _require_cuda(x, w13, w2, group_sizes)
    _check_shapes(x, w13, w2)
    E, H, inter, group, a, sa, b, sb = _layer_weights(x, w13, w2, w13_scale, w2_scale)
    dev = _one_device("fused_moe_mlp", x, w13, w2, group_sizes, w13_scale, w2_scale)
    x = x.contiguous()
    _check_counts("fused_moe_mlp", group_sizes, E)
    gs = _counts(group_sizes)
    T = x.shape[0]
    out = torch.empty((T, H), dtype=x.dtype, device=dev)
    size = _lib.query("moe_fused_mlp_int4_workspace_size", T, inter, E)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _launch(dev, "moe_fused_mlp_int4", x.data_ptr(), _CODES[x.dtype], T, H, a.data_ptr(), sa.data_ptr(), b.data_ptr(),
            sb.data_ptr(), group, E, inter, gs.data_ptr(), _lib.I32 if gs.dtype == torch.int32 else _lib.I64,
            out.data_ptr(), ws.data_ptr(), size)
    return out


@torch.library.custom_op("mail_b200::fused_moe_mlp_int4", mutates_args=())
def _op_prerouted(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, group_sizes: torch.Tensor,
                  w13_scale: torch.Tensor, w2_scale: torch.Tensor) -> torch.Tensor:
    return fused_mlp(x, w13, w2, group_sizes, w13_scale, w2_scale)


@_op_prerouted.register_fake
def _(x, w13, w2, group_sizes, w13_scale, w2_scale):
    T, H, E, _ = _check_shapes(x, w13, w2)
    check_layer(x, w13, w2, w13_scale, w2_scale)
    _check_counts("fused_moe_mlp", group_sizes, E)
    return x.new_empty((T, H))


@torch.library.custom_op("mail_b200::grouped_matmul_int4", mutates_args=())
def _op_grouped(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, group_sizes: torch.Tensor) -> torch.Tensor:
    return _grouped_impl(x, w, scale, group_sizes)


@_op_grouped.register_fake
def _(x, w, scale, group_sizes):
    _check_grouped(x, w, scale, group_sizes)
    return x.new_empty((x.shape[0], w.shape[2]))
