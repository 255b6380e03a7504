"""Cases that measure the linear products and the 8-bit block quantizers of quant_2bit_b200.

Four operators, the shapes of the layers that the framework quantizes (projections of 2048, 8192 and
512 features, layers of 64 experts with 2048 and 1024 features) and generic sizes between them:

* ``quantize``  a matrix in e4m3 with one fp32 scale for each 1 x 128 row segment (activations) or
  each 128 x 128 block (weights);
* ``fp8``       a linear layer over such a weight: activations quantized by row segments, products
  summed in fp32, and the gradient of the activations;
* ``grouped``   rows sorted by expert times each expert's weight, ragged group sizes, with both
  gradients;
* ``fp8 experts``  ``fp8`` with one weight for each group of rows.

``own`` False computes the plain form with elementary torch operations in fp32, True calls the
framework.
"""
import math

import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
AMAX_MIN = 2.0 ** -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token's activations before an 8-bit projection: latency
        {"name": "quantize_row_one_token", "op": "quantize", "blocks": False, "rows": 1, "k": 2048,
         "dtype": "bf16"},
        # a down projection's fp32 master weight, quantized when a model is loaded
        {"name": "quantize_weight_2048x8192", "op": "quantize", "blocks": True, "rows": 2048,
         "k": 8192, "dtype": "fp32"},
        # one generated token through an up projection
        {"name": "fp8_one_token", "op": "fp8", "rows": 1, "n": 8192, "k": 2048, "experts": 0,
         "top_k": 0, "dtype": "bf16", "backward": False},
        # 37 sequences that each generate a token, down projection
        {"name": "fp8_batch_37", "op": "fp8", "rows": 37, "n": 2048, "k": 8192, "experts": 0,
         "top_k": 0, "dtype": "fp16", "backward": False},
        # a prompt batch of 8192 tokens
        {"name": "fp8_prompt_8192", "op": "fp8", "rows": 8192, "n": 8192, "k": 2048, "experts": 0,
         "top_k": 0, "dtype": "bf16", "backward": False},
        # a frozen 8-bit layer inside a network that trains: odd token count, widths that end
        # inside a block of 128, and the gradient that flows through it
        {"name": "fp8_frozen_layer_1237", "op": "fp8", "rows": 1237, "n": 2000, "k": 2128,
         "experts": 0, "top_k": 0, "dtype": "bf16", "backward": True},
        # 8-bit experts, 16 tokens generated at once
        {"name": "fp8_experts_16_tokens", "op": "fp8", "rows": 16, "n": 1024, "k": 2048,
         "experts": 64, "top_k": 8, "dtype": "bf16", "backward": False},
        # 8-bit experts, a prompt of 4096 tokens
        {"name": "fp8_experts_4096_tokens", "op": "fp8", "rows": 4096, "n": 2048, "k": 1024,
         "experts": 64, "top_k": 8, "dtype": "bf16", "backward": False},
        # one generated token through its 8 experts
        {"name": "grouped_one_token", "op": "grouped", "rows": 1, "n": 1024, "k": 2048,
         "experts": 64, "top_k": 8, "dtype": "bf16", "backward": False, "pad": 0},
        # 61 tokens generated at once, down projection of the experts
        {"name": "grouped_61_tokens", "op": "grouped", "rows": 61, "n": 2048, "k": 1024,
         "experts": 64, "top_k": 8, "dtype": "fp16", "backward": False, "pad": 0},
        # a small layer that trains: odd sizes, empty groups, padding rows behind the last group
        {"name": "grouped_train_ragged", "op": "grouped", "rows": 1501, "n": 528, "k": 272,
         "experts": 96, "top_k": 2, "dtype": "fp16", "backward": True, "pad": 77},
        # the training step of the 64-expert layer: 4096 tokens, forward and both gradients
        {"name": "grouped_train_4096_tokens", "op": "grouped", "rows": 4096, "n": 1024, "k": 2048,
         "experts": 64, "top_k": 8, "dtype": "bf16", "backward": True, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    return max(lo, 16 * (_log(rng, lo, hi) // 16))


def draw(rng):
    op = rng.choice(["quantize", "fp8", "fp8", "experts", "grouped", "grouped"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "quantize":
        return {"op": op, "blocks": rng.random() < 0.5, "rows": _log(rng, 1, 8192),
                "k": _width(rng, 16, 8192), "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    backward = rng.random() < 0.5
    if op == "fp8":
        rows = _log(rng, 1, 8192)
        n, k = _width(rng, 128, 8192), _width(rng, 128, 8192)
        while rows * n * k * (2 if backward else 1) > 8192 * 8192 * 2048:
            rows //= 2
        return {"op": op, "rows": rows, "n": n, "k": k, "experts": 0, "top_k": 0, "dtype": dtype,
                "backward": backward}
    experts = _log(rng, 2, 128)
    top_k = rng.randint(1, min(8, experts))
    n, k = _width(rng, 64, 2048), _width(rng, 64, 2048)
    rows = _log(rng, 1, 4096)
    while rows * top_k * n * k > 4096 * 8 * 1024 * 2048 or rows * top_k * max(n, k) > 4096 * 8 * 2048:
        rows //= 2
    case = {"rows": rows, "n": n, "k": k, "experts": experts, "top_k": top_k, "dtype": dtype,
            "backward": backward}
    if op == "experts":
        return {"op": "fp8", **case}
    return {"op": "grouped", **case, "pad": rng.choice([0, 0, rng.randint(1, 200)])}


def _pad128(v):
    return -(-v // 128) * 128


def _amax_to_scale(amax):
    """(scale, its reciprocal's stand-in) of a block: x is stored as the e4m3 nearest to x * inv."""
    amax = amax.clamp(min=AMAX_MIN)
    return amax / F8_MAX, F8_MAX / amax


def _quantize_rows(x):
    """e4m3 values and the (rows, ceil(k / 128)) scales of row segments of 128."""
    rows, k = x.shape
    xb = torch.nn.functional.pad(x.float(), (0, _pad128(k) - k)).view(rows, -1, 128)
    scale, inv = _amax_to_scale(xb.abs().amax(-1))
    q = (xb * inv.unsqueeze(-1)).to(F8).view(rows, -1)[:, :k]
    return q.contiguous(), scale


def _quantize_blocks(w):
    """e4m3 values and the (ceil(n / 128), ceil(k / 128)) scales of 128 x 128 blocks (last two axes)."""
    n, k = w.shape[-2:]
    lead = w.shape[:-2]
    wb = torch.nn.functional.pad(w.float(), (0, _pad128(k) - k, 0, _pad128(n) - n))
    wb = wb.view(*lead, _pad128(n) // 128, 128, _pad128(k) // 128, 128)
    scale, inv = _amax_to_scale(wb.abs().amax(-1).amax(-2))
    q = (wb * inv[..., :, None, :, None]).to(F8).view(*lead, _pad128(n), _pad128(k))[..., :n, :k]
    return q.contiguous(), scale


def _expand_rows(q, scale):
    return q.float() * scale.repeat_interleave(128, dim=-1)[..., :q.shape[-1]]


def _expand_blocks(q, scale):
    s = scale.repeat_interleave(128, dim=-1)[..., :q.shape[-1]]
    return q.float() * s.repeat_interleave(128, dim=-2)[..., :q.shape[-2], :]


def _activations(rows, k, gen, scale=1.0):
    """Normal values with a few channels that are much larger, as activations have them."""
    x = torch.randn(rows, k, generator=gen, device="cuda") * scale
    loud = torch.randint(0, k, (max(1, k // 256),), generator=gen, device="cuda")
    x[:, loud] *= 12.0
    return x


def _route(rows, experts, top_k, gen):
    """Rows of each expert: every token picks its top_k of unequally liked experts."""
    liked = 0.5 * torch.randn(experts, generator=gen, device="cuda")
    noise = torch.rand(rows, experts, generator=gen, device="cuda").clamp_(1e-6, 1 - 1e-6)
    pick = (liked - torch.log(-torch.log(noise))).topk(top_k, dim=-1).indices
    counts = torch.bincount(pick.reshape(-1), minlength=experts)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return offsets, int(counts.max())


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "quantize":
        if case["blocks"]:
            s["x"] = (0.02 * torch.randn(case["rows"], case["k"], generator=gen, device="cuda")).to(dtype)
        else:
            s["x"] = _activations(case["rows"], case["k"], gen).to(dtype)
        return s
    n, k, experts = case["n"], case["k"], case["experts"]
    rows, s["offsets"], s["cap"] = case["rows"], None, None
    if experts:
        s["offsets"], s["cap"] = _route(rows, experts, case["top_k"], gen)
        rows = rows * case["top_k"] + case.get("pad", 0)
    x = _activations(rows, k, gen).to(dtype)
    shape = (experts, n, k) if experts else (n, k)
    w = torch.randn(shape, generator=gen, device="cuda") / math.sqrt(k)
    if case["op"] == "fp8":
        s["q"], s["scale"] = _quantize_blocks(w)
    else:
        s["w"] = w.to(dtype).requires_grad_(case["backward"])
    if case["backward"]:
        s["dy"] = (0.01 * torch.randn(rows, n, generator=gen, device="cuda")).to(dtype)
    s["x"] = x.requires_grad_(case["backward"])
    return s


def _places(offsets, rows, cap):
    """Where each row goes in an (experts, cap) table; rows of no group go behind its end."""
    experts = offsets.numel() - 1
    row = torch.arange(rows, device=offsets.device)
    e = torch.searchsorted(offsets[1:].contiguous(), row.to(offsets.dtype), right=True)
    first = offsets[:-1].long()[e.clamp(max=experts - 1)]
    return torch.where(e < experts, e * cap + row - first, experts * cap)


def _to_table(x, place, experts, cap):
    t = torch.zeros(experts * cap + 1, x.shape[1], device=x.device)
    t[place] = x.float()
    return t[:-1].view(experts, cap, -1)


def _from_table(t, place):
    flat = t.reshape(-1, t.shape[-1])
    return torch.cat([flat, flat.new_zeros(1, flat.shape[1])])[place]


def _rows_times(x, w, offsets, cap):
    """x's rows times the transpose of their group's w (or of the only one), fp32."""
    if offsets is None:
        return x.float() @ w.t()
    place = _places(offsets, x.shape[0], cap)
    return _from_table(torch.bmm(_to_table(x, place, w.shape[0], cap), w.transpose(1, 2)), place)


def _plain(s):
    x = s["x"].detach()
    if s["op"] == "quantize":
        return (_quantize_blocks if s["blocks"] else _quantize_rows)(x)
    offsets, cap = s["offsets"], s["cap"]
    if s["op"] == "fp8":
        w = _expand_blocks(s["q"], s["scale"])
        y = _rows_times(_expand_rows(*_quantize_rows(x)), w, offsets, cap).to(x.dtype)
        if not s["backward"]:
            return {"y": y}
        g = _expand_rows(*_quantize_rows(s["dy"]))
        return {"y": y, "dx": _rows_times(g, w.transpose(-1, -2), offsets, cap).to(x.dtype)}
    w = s["w"].detach().float()
    y = _rows_times(x, w, offsets, cap).to(x.dtype)
    if not s["backward"]:
        return {"y": y}
    dy = s["dy"]
    dx = _rows_times(dy, w.transpose(1, 2), offsets, cap).to(x.dtype)
    place = _places(offsets, x.shape[0], cap)
    dw = torch.bmm(_to_table(dy, place, w.shape[0], cap).transpose(1, 2),
                   _to_table(x, place, w.shape[0], cap))
    return {"y": y, "dx": dx, "dw": dw.to(x.dtype)}


def run(state):
    s = state
    if not own:
        return _plain(s)
    from quant_2bit_b200 import fp8_linear, fp8_quantize_rows, fp8_quantize_weight, grouped_linear
    if s["op"] == "quantize":
        return fp8_quantize_weight(s["x"]) if s["blocks"] else fp8_quantize_rows(s["x"])
    if s["op"] == "fp8":
        y = fp8_linear(s["x"], s["q"], s["scale"], offsets=s["offsets"])
        if not s["backward"]:
            return {"y": y}
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    y = grouped_linear(s["x"], s["w"], s["offsets"])
    if not s["backward"]:
        return {"y": y}
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "quantize":
        cells = case["rows"] * case["k"]
        segments = -(-case["k"] // 128) * (-(-case["rows"] // 128) if case["blocks"] else case["rows"])
        return {"bytes": cells * (size + 1) + 4 * segments, "flops": 3 * cells}
    n, k = case["n"], case["k"]
    rows = case["rows"] * max(1, case["top_k"])
    weights = n * k * min(max(1, case["experts"]), rows)
    io = rows * (n + k) * size
    flops = 2 * rows * n * k
    passes = 2 if case["backward"] else 1
    if case["op"] == "fp8":
        return {"bytes": passes * (io + weights + 4 * weights // 16384), "flops": passes * flops}
    if not case["backward"]:
        return {"bytes": io + weights * size, "flops": flops}
    # x, dy, w read; y, dx, dw written (dw also for experts without rows)
    return {"bytes": 2 * io + (weights + n * k * case["experts"]) * size, "flops": 3 * flops}


def _codes64(x, rows_of_block):
    """The stored values in 64 bits, code times scale: block maxima, the scale and the scaled value
    are fp32 by definition, so they are formed in fp32 here too, block by block."""
    n, k = x.shape
    out = torch.empty(n, k, dtype=torch.float64, device=x.device)
    codes = torch.empty(n, k, dtype=torch.float64, device=x.device)
    scales = torch.empty(-(-n // rows_of_block), -(-k // 128), dtype=torch.float64, device=x.device)
    for j in range(0, k, 128):
        strip = x[:, j:j + 128].to(torch.float32)
        top = strip.abs().max(dim=1).values
        if rows_of_block > 1:
            top = torch.stack([t.max() for t in top.split(rows_of_block)])
        top = torch.maximum(top, torch.full_like(top, AMAX_MIN))
        each = torch.repeat_interleave(top, rows_of_block)[:n, None]
        code = (strip * (F8_MAX / each)).to(F8).double()
        codes[:, j:j + 128] = code
        out[:, j:j + 128] = code * (each / F8_MAX).double()
        scales[:, j // 128] = (top / F8_MAX).double()
    return codes, scales, out


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach()
    if case["op"] == "quantize":
        codes, scales, _ = _codes64(x, 128 if case["blocks"] else 1)
        return codes, scales
    if case["op"] == "fp8":
        w = s["q"].double()
        blocks = s["scale"].double()
        at_n = torch.arange(w.shape[-2], device=w.device) // 128
        at_k = torch.arange(w.shape[-1], device=w.device) // 128
        w = w * blocks[..., at_n, :][..., at_k]
        a = _codes64(x, 1)[2]
        g = _codes64(s["dy"], 1)[2] if case["backward"] else None
    else:
        w, a = s["w"].detach().double(), x.double()
        g = s["dy"].double() if case["backward"] else None
    w = w if w.dim() == 3 else w.unsqueeze(0)
    ends = [0, x.shape[0]] if s["offsets"] is None else s["offsets"].tolist()
    y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=x.device)
    dx = torch.zeros(x.shape[0], case["k"], dtype=torch.float64, device=x.device)
    dw = torch.zeros_like(w) if case["op"] == "grouped" and case["backward"] else None
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if hi > lo:
            y[lo:hi] = torch.einsum("tk,nk->tn", a[lo:hi], w[e])
            if g is not None:
                dx[lo:hi] = torch.einsum("tn,nk->tk", g[lo:hi], w[e])
            if dw is not None:
                dw[e] = torch.einsum("tn,tk->nk", g[lo:hi], a[lo:hi])
    out = {"y": y}
    if g is not None:
        out["dx"] = dx
    if dw is not None:
        out["dw"] = dw
    return out
