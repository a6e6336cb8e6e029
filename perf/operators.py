"""The 4-bit expert operators as measured cases: quantising weights to 4 bits
with group scales and reading them back, the matrix product grouped by expert,
and the whole expert layer, each in a plain torch form and as the framework's
call.

A packed weight is uint8 [N, K / 2] for each expert: byte b of a row holds
element 2b in its low and 2b + 1 in its high nibble, element q stands for
(q - 8) * scale[n, k // group].
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MAX_FLOPS = 3.0e12     # a drawn case stays below the largest listed ones
_MAX_WEIGHTS = 3.0e9    # 4-bit weights of a drawn case
_MAX_QUANT = 4.6e8      # weights quantised in a drawn case


def listed():
    return [
        # one expert's gate and up weights, quantised as a checkpoint loads
        {"name": "quant-expert", "op": "quant", "R": 1536, "C": 2048, "group": 128, "dtype": "bf16"},
        # the down weights of a whole layer of eight large experts, the fine groups
        {"name": "quant-layer", "op": "quant", "R": 32768, "C": 14336, "group": 32, "dtype": "bf16"},
        # a single token's two rows through the gate and up weights: pure weight streaming
        {"name": "grouped-token", "op": "grouped", "T": 2, "K": 4096, "N": 28672, "E": 8, "group": 128,
         "dtype": "bf16", "skew": 0.0},
        # a decode batch over many small experts, some of them popular
        {"name": "grouped-decode", "op": "grouped", "T": 256, "K": 2048, "N": 1536, "E": 128, "group": 128,
         "dtype": "bf16", "skew": 0.7},
        # odd and ragged sizes in fp16: N odd, K no multiple of 64, few experts of uneven size
        {"name": "grouped-odd", "op": "grouped", "T": 777, "K": 1056, "N": 1001, "E": 5, "group": 32,
         "dtype": "fp16", "skew": 1.0},
        # prefill over eight large experts: bound by the tensor cores
        {"name": "grouped-prefill", "op": "grouped", "T": 8192, "K": 4096, "N": 14336, "E": 8, "group": 128,
         "dtype": "bf16", "skew": 0.1},
        # one token through the layer of many small experts: latency
        {"name": "layer-small-1", "op": "layer", "T": 1, "H": 2048, "I": 768, "E": 128, "k": 8, "group": 128,
         "dtype": "bf16", "skew": 0.0},
        # one token through the layer of few large experts: weight streaming
        {"name": "layer-large-1", "op": "layer", "T": 1, "H": 4096, "I": 14336, "E": 8, "k": 2, "group": 128,
         "dtype": "bf16", "skew": 0.0},
        # decode batches of the small-expert layer, fp16 and the finer groups among them
        {"name": "layer-small-16", "op": "layer", "T": 16, "H": 2048, "I": 768, "E": 128, "k": 8, "group": 64,
         "dtype": "fp16", "skew": 0.5},
        {"name": "layer-small-256", "op": "layer", "T": 256, "H": 2048, "I": 768, "E": 128, "k": 8, "group": 128,
         "dtype": "bf16", "skew": 0.3},
        # a prefill chunk over 256 experts, 32 rows an expert: between the two bounds
        {"name": "layer-many-1024", "op": "layer", "T": 1024, "H": 7168, "I": 2048, "E": 256, "k": 8, "group": 128,
         "dtype": "bf16", "skew": 0.2},
        # prefill of the large-expert layer
        {"name": "layer-large-4096", "op": "layer", "T": 4096, "H": 4096, "I": 14336, "E": 8, "k": 2, "group": 128,
         "dtype": "bf16", "skew": 0.1},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["quant", "grouped", "grouped", "layer", "layer"])
    group = rng.choice([32, 64, 128])
    while True:
        if op == "quant":
            case = {"op": op, "R": _log_int(rng, 1, 40000), "C": group * _log_int(rng, 1, 14336 // group),
                    "group": group, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
            if case["R"] * case["C"] <= _MAX_QUANT:
                return case
        elif op == "grouped":
            case = {"op": op, "T": _log_int(rng, 1, 8192), "K": group * _log_int(rng, 1, 7168 // group),
                    "N": _log_int(rng, 1, 28672), "E": _log_int(rng, 1, 256), "group": group,
                    "dtype": rng.choice(["bf16", "fp16"]), "skew": rng.choice([0.0, 0.3, 0.7, 1.0])}
            if (2.0 * case["T"] * case["K"] * case["N"] <= _MAX_FLOPS / 3
                    and case["E"] * case["K"] * case["N"] <= _MAX_WEIGHTS):
                return case
        else:
            E = _log_int(rng, 1, 256)
            case = {"op": op, "T": _log_int(rng, 1, 4096), "H": group * _log_int(rng, 1, 7168 // group),
                    "I": group * _log_int(rng, 1, 14336 // group), "E": E, "k": rng.randint(1, min(8, E)),
                    "group": group, "dtype": rng.choice(["bf16", "fp16"]), "skew": rng.choice([0.0, 0.2, 0.5])}
            if (6.0 * case["T"] * case["k"] * case["H"] * case["I"] <= _MAX_FLOPS * 0.9
                    and 3 * E * case["H"] * case["I"] <= _MAX_WEIGHTS):
                return case


# ------------------------------------------------------------------- inputs


def _popularity(E, skew):
    """How often each expert is hit: 1 / rank ** skew, normalised."""
    p = [(e + 1.0) ** -skew for e in range(E)]
    s = sum(p)
    return [v / s for v in p]


def _packed_weights(E, N, K, group, dtype, gen):
    """4-bit weights as quantising normal weights gives them: a bell over the
    16 values, scales near 0.4 of a standard deviation that fits the fan-in."""
    packed = torch.empty((E, N, K // 2), dtype=torch.uint8, device="cuda")
    for e in range(E):
        q = torch.randn((N, K), device="cuda", generator=gen).mul_(2.4).add_(8.0).round_().clamp_(0, 15)
        q = q.to(torch.uint8)
        packed[e] = q[:, 0::2] | (q[:, 1::2] << 4)
    scale = torch.rand((E, N, K // group), device="cuda", generator=gen).add_(0.5).mul_(0.42 / math.sqrt(K))
    return packed, scale.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    st = {"op": case["op"], "group": case["group"]}
    if case["op"] == "quant":
        w = torch.empty((case["R"], case["C"]), dtype=dtype, device="cuda")
        for i in range(0, case["R"], 4096):
            part = w[i:i + 4096]
            part.copy_(torch.randn(part.shape, device="cuda", generator=gen).mul_(0.02))
        st["w"] = w
    elif case["op"] == "grouped":
        p = torch.tensor(_popularity(case["E"], case["skew"]), device="cuda")
        p = p[torch.randperm(case["E"], device="cuda", generator=gen)]
        rows = torch.multinomial(p, case["T"], replacement=True, generator=gen)
        st["group_sizes"] = torch.bincount(rows, minlength=case["E"]).to(torch.int32)
        st["x"] = torch.randn((case["T"], case["K"]), device="cuda", generator=gen).to(dtype)
        packed, st["scale"] = _packed_weights(case["E"], case["N"], case["K"], case["group"], dtype, gen)
        st["w"] = packed.transpose(1, 2)
    else:
        T, H, I, E, k = case["T"], case["H"], case["I"], case["E"], case["k"]
        p = torch.tensor(_popularity(E, case["skew"]), device="cuda")
        p = p[torch.randperm(E, device="cuda", generator=gen)]
        gumbel = -torch.log(-torch.log(torch.rand((T, E), device="cuda", generator=gen).clamp_(1e-6, 1 - 1e-6)))
        top = torch.topk(gumbel + torch.log(p), k, dim=1)
        st["ids"] = top.indices.to(torch.int32)
        st["weights"] = torch.softmax(top.values, dim=1).float()
        st["x"] = torch.randn((T, H), device="cuda", generator=gen).to(dtype)
        w13, st["s13"] = _packed_weights(E, 2 * I, H, case["group"], dtype, gen)
        w2, st["s2"] = _packed_weights(E, H, I, case["group"], dtype, gen)
        st["w13"], st["w2"] = w13.transpose(1, 2), w2.transpose(1, 2)
    return st


# --------------------------------------------------------------- plain form


def _values(packed, scale, group):
    """Packed rows [N, K / 2] and scales [N, K / group] -> fp32 weights [N, K]."""
    N, half = packed.shape
    q = torch.stack((packed & 15, packed >> 4), dim=-1).view(N, 2 * half // group, group)
    return ((q.float() - 8.0) * scale.float().unsqueeze(-1)).view(N, 2 * half)


def _plain_quant(w, group):
    """s = absmax / 7 rounded to the scales' type, q = x / s rounded half to
    even and clamped; the quotient in 64 bits, where no border moves. Returns
    the values that the 4 bits stand for, and the scales."""
    R, C = w.shape
    stype = w.dtype if w.dtype != torch.float32 else torch.bfloat16
    values = torch.empty_like(w)
    scales = torch.empty((R, C // group), dtype=stype, device=w.device)
    step = max(1, (1 << 25) // C)
    for i in range(0, R, step):
        part = w[i:i + step].float().view(-1, C // group, group)
        s = (part.abs().amax(dim=-1) / 7.0).to(stype)
        sd = s.double().unsqueeze(-1)
        q = torch.where(sd > 0, part.double() / sd, torch.zeros((), dtype=torch.float64, device=w.device))
        q = torch.round(q).clamp(-8, 7).float()
        values[i:i + step] = (q * s.float().unsqueeze(-1)).view(-1, C).to(w.dtype)
        scales[i:i + step] = s
    return values, scales


def _picked(w, scale, ids, group):
    """The fp32 weights [S, N, K] of the experts that S rows name."""
    E, N, half = w.shape
    picked = _values(w[ids].reshape(-1, half), scale[ids].reshape(-1, scale.shape[2]), group)
    return picked.view(-1, N, 2 * half)


def _plain_grouped(st):
    x, w, scale = st["x"], st["w"].transpose(1, 2), st["scale"]
    if x.shape[0] <= 8:  # a few rows: their experts' weights at once
        ends = torch.cumsum(st["group_sizes"], 0)
        ids = torch.searchsorted(ends, torch.arange(x.shape[0], device=x.device), right=True)
        return torch.bmm(_picked(w, scale, ids, st["group"]), x.float().unsqueeze(-1)).squeeze(-1).to(x.dtype)
    out = torch.zeros((x.shape[0], w.shape[1]), dtype=x.dtype, device=x.device)
    row = 0
    for e, n in enumerate(st["group_sizes"].tolist()):
        if n:
            out[row:row + n] = (x[row:row + n].float() @ _values(w[e], scale[e], st["group"]).t()).to(x.dtype)
        row += n
    return out


def _plain_layer(st):
    x, ids, weights = st["x"], st["ids"], st["weights"]
    w13, w2 = st["w13"].transpose(1, 2), st["w2"].transpose(1, 2)
    T, k = ids.shape
    inter = w13.shape[1] // 2
    flat = ids.flatten()
    if T * k <= 8:  # a few slots: their experts' weights at once
        rows = x.float().repeat_interleave(k, dim=0).unsqueeze(-1)
        g, u = torch.bmm(_picked(w13, st["s13"], flat, st["group"]), rows).split(inter, dim=1)
        o = torch.bmm(_picked(w2, st["s2"], flat, st["group"]), g / (1.0 + torch.exp(-g)) * u)
        return (o.view(T, k, -1) * weights.unsqueeze(-1)).sum(dim=1).to(x.dtype)
    order = torch.argsort(flat, stable=True)
    slots = torch.empty((T * k, x.shape[1]), dtype=torch.float32, device=x.device)
    row = 0
    for e, n in enumerate(torch.bincount(flat, minlength=w13.shape[0]).tolist()):
        if n:
            mine = order[row:row + n]
            gu = x[mine // k].float() @ _values(w13[e], st["s13"][e], st["group"]).t()
            g, u = gu[:, :inter], gu[:, inter:]
            h = g / (1.0 + torch.exp(-g)) * u
            slots[mine] = h @ _values(w2[e], st["s2"][e], st["group"]).t()
        row += n
    return (slots.view(T, k, -1) * weights.unsqueeze(-1)).sum(dim=1).to(x.dtype)


# ------------------------------------------------------------------ the run


def run(st):
    if own:
        import mail_b200 as mb

        if st["op"] == "quant":
            q, s = mb.quant_int4_groups(st["w"], group_size=st["group"])
            return mb.dequant_int4_groups(q, s, dtype=st["w"].dtype), s
        if st["op"] == "grouped":
            return mb.grouped_matmul_int4(st["x"], st["w"], st["scale"], st["group_sizes"])
        return mb.fused_moe_mlp(st["x"], st["w13"], st["w2"], st["weights"], st["ids"], scales=(st["s13"], st["s2"]))
    if st["op"] == "quant":
        return _plain_quant(st["w"], st["group"])
    if st["op"] == "grouped":
        return _plain_grouped(st)
    return _plain_layer(st)


def _hit(E, skew, picks):
    """Experts that `picks` picks are expected to hit."""
    return sum(-math.expm1(picks * math.log1p(-min(p, 1 - 1e-12))) for p in _popularity(E, skew))


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "quant":
        n = case["R"] * case["C"]
        return {"bytes": 2 * es * n + 2 * n // case["group"], "flops": 4 * n}
    per_weight = 0.5 + 2.0 / case["group"]
    if case["op"] == "grouped":
        T, K, N = case["T"], case["K"], case["N"]
        weights = _hit(case["E"], case["skew"], T) * K * N * per_weight
        return {"bytes": int(weights + 2 * T * (K + N) + 4 * case["E"]), "flops": 2 * T * K * N}
    T, H, I, k = case["T"], case["H"], case["I"], case["k"]
    weights = max(_hit(case["E"], case["skew"], T * k), min(k, case["E"])) * 3 * H * I * per_weight
    return {"bytes": int(weights + 4 * T * H + 8 * T * k), "flops": 6 * T * k * H * I}


# ------------------------------------------------------- 64-bit definitions


def _wide(packed, scale, group):
    """The weights [N, K] in 64 bits, from the bytes by division."""
    n, half = packed.shape
    out = torch.empty((n, 2 * half), dtype=torch.float64, device=packed.device)
    b = packed.to(torch.float64)
    high = torch.floor(b / 16.0)
    out[:, 1::2] = high - 8.0
    out[:, 0::2] = b - 16.0 * high - 8.0
    return out * torch.repeat_interleave(scale.double(), group, dim=1)


def exact(case, seed):
    st = prepare(case, seed)
    group = st["group"]
    if case["op"] == "quant":
        w = st["w"]
        stype = torch.bfloat16 if w.dtype == torch.float32 else w.dtype
        values = torch.empty(w.shape, dtype=torch.float64, device=w.device)
        scales = torch.empty((w.shape[0], w.shape[1] // group), dtype=torch.float64, device=w.device)
        for g in range(w.shape[1] // group):
            cols = w[:, g * group:(g + 1) * group].double()
            s = (cols.abs().max(dim=1, keepdim=True).values / 7.0).float().to(stype).double()
            q = torch.minimum(torch.maximum(torch.round(cols / s.clamp_min(1e-300)), -8 * torch.ones_like(s)),
                              7 * torch.ones_like(s))
            values[:, g * group:(g + 1) * group] = q * s
            scales[:, g:g + 1] = s
        return values, scales
    x = st["x"].double()
    if case["op"] == "grouped":
        ends = torch.cumsum(st["group_sizes"], 0).tolist()
        out = torch.zeros((case["T"], case["N"]), dtype=torch.float64, device=x.device)
        start = 0
        for e, end in enumerate(ends):
            if end > start:
                wide = _wide(st["w"][e].t(), st["scale"][e], group)
                out[start:end] = torch.mm(x[start:end], wide.t())
            start = end
        return out
    y = torch.zeros((case["T"], case["H"]), dtype=torch.float64, device=x.device)
    inter = case["I"]
    for e in range(case["E"]):
        tok, col = torch.nonzero(st["ids"] == e, as_tuple=True)
        if tok.numel() == 0:
            continue
        up_gate = _wide(st["w13"][e].t(), st["s13"][e], group)
        rows = x[tok]
        gate = torch.mm(rows, up_gate[:inter].t())
        h = gate * torch.sigmoid(gate) * torch.mm(rows, up_gate[inter:].t())
        o = torch.mm(h, _wide(st["w2"][e].t(), st["s2"][e], group).t())
        y.index_add_(0, tok, o * st["weights"][tok, col].double().unsqueeze(1))
    return y
