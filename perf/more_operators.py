"""Cases of the microscaled 4-bit products and of the whole mixture-of-experts
layer: f16acc_amd.fp4 and f16acc_amd.moe.layer.

"quantize"  fp4.quantize(x) and fp4.dequantize of it: activations to blocks of 32
            4-bit values with a power of two each, and the values that they stand for.
"mm"        fp4.mm(a, a_scale, b, b_scale, out_dtype) of stored operands.
"linear"    fp4.linear(x, w, w_scale, bias): 16- or 32-bit activations quantised on
            the way, times a stored 4-bit weight.
"train"     the same layer on a 16-bit weight, forward and backward: y, dx, dw, each
            product's operands quantised along its own sum.
"layer"     moe.layer(x, router, k, w1, ...): router product, choice of k experts,
            and the experts' gated FFN in 8 bits (blocks of 128).

A block of 32 is held as s = 2^e with 2^e <= m / 3.5 < 2^(e + 1), m = max(|x|, 2^-100),
and the e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) nearest to x / s, ties to
the even code.  Two values share a byte, the first in its low half.
"""

import math

import torch

# False: run() computes the plain forms below.  True: it calls the framework.
own = False

DEV = "cuda"
MX = 32      # values of a 4-bit block
BLOCK = 128  # values of an 8-bit block
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # Activations of a short batch whose width ends inside a block and a byte.
        dict(name="quantize_odd_77", op="quantize", M=77, K=8961, type="bf16"),
        # The activations of a long prompt, at the width of the largest product.
        dict(name="quantize_8192", op="quantize", M=8192, K=8192, type="bf16"),
        # A short ragged product of stored operands, FP32 result.
        dict(name="mm_odd_200", op="mm", M=200, N=1537, K=8962, out="f32"),
        # Qwen2.5-1.5B's gate/up layer over a prompt of 2048 tokens, operands quantised already.
        dict(name="mm_gateup_2048", op="mm", M=2048, N=8960, K=1536, out="bf16"),
        # One token through that layer: a decode step, which reads the weight.
        dict(name="linear_token", op="linear", M=1, N=8960, K=1536, type="f16", bias=False),
        # A short batch against a weight whose rows no 16-byte load fits.
        dict(name="linear_odd_77", op="linear", M=77, N=1537, K=8961, type="bf16", bias=True),
        # The largest product: the square the 16-bit GEMM is measured on.
        dict(name="linear_8192", op="linear", M=8192, N=8192, K=8192, type="bf16", bias=False),
        # Training steps of the q/o projection and of the down projection.
        dict(name="train_qo_2048", op="train", M=2048, N=1536, K=1536, type="bf16"),
        dict(name="train_down_4096", op="train", M=4096, N=1536, K=8960, type="f16"),
        # A decode step of one sequence through a mixture of 64 experts.
        dict(name="layer_token", op="layer", T=1, E=64, k=6, D=2048, I=1024, type="f16", scoring="softmax", bias=False,
             groups=1, top=1, renormalize=True, router="f16"),
        # Three sequences; widths that end inside a block, a balance bias, groups, an FP32 router.
        dict(name="layer_odd_3", op="layer", T=3, E=20, k=4, D=1040, I=720, type="bf16", scoring="sigmoid", bias=True,
             groups=4, top=2, renormalize=True, router="f32"),
        # A prompt of 512 tokens, past what the kernels for a few tokens take.
        dict(name="layer_512", op="layer", T=512, E=64, k=8, D=2048, I=1024, type="bf16", scoring="softmax", bias=False,
             groups=1, top=1, renormalize=True, router="bf16"),
    ]


def _extent(rng, lo, hi, odd=0.15):
    """An extent spread over its logarithm: mostly multiples of 128, else of
    16, else any number."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    r = rng.random()
    step = 1 if r < odd else 16 if r < 0.4 else 128
    return max(lo, min(hi, v // step * step))


def draw(rng):
    op = rng.choice(["quantize", "mm", "linear", "linear", "train", "layer", "layer"])
    while True:
        if op == "quantize":
            c = dict(op=op, M=_extent(rng, 1, 8192, odd=0.6), K=_extent(rng, 32, 12288, odd=0.4),
                     type=rng.choice(["f16", "bf16", "f32"]))
            cost = 0
        elif op == "mm":
            c = dict(op=op, M=_extent(rng, 1, 8192, odd=0.6), N=_extent(rng, 128, 16384),
                     K=2 * _extent(rng, 64, 6144), out=rng.choice(["f16", "bf16", "f32"]))
            cost = c["M"] * c["N"] * c["K"]
        elif op == "linear":
            c = dict(op=op, M=_extent(rng, 1, 8192, odd=0.6), N=_extent(rng, 128, 16384), K=_extent(rng, 128, 12288),
                     type=rng.choice(["f16", "bf16", "bf16", "f32"]), bias=rng.random() < 0.5)
            cost = c["M"] * c["N"] * c["K"]
        elif op == "train":
            c = dict(op=op, M=_extent(rng, 128, 8192), N=_extent(rng, 128, 8960), K=_extent(rng, 128, 8960),
                     type=rng.choice(["f16", "bf16"]))
            cost = 3 * c["M"] * c["N"] * c["K"]
        else:
            groups = rng.choice([1, 1, 4, 8])
            E = groups * rng.randint(max(1, 8 // groups), 128 // groups)
            top = rng.randint(1, groups)
            kind = rng.choice(["f16", "bf16"])
            c = dict(op=op, T=rng.choice([1, 1, 2, 3, 4, _extent(rng, 5, 1024, odd=0.8)]), E=E,
                     k=rng.randint(1, min(8, top * E // groups)), D=_extent(rng, 256, 4096, odd=0.0),
                     I=_extent(rng, 256, 2048, odd=0.0), type=kind, scoring=rng.choice(["softmax", "sigmoid"]),
                     bias=False, groups=groups, top=top, renormalize=rng.random() < 0.7,
                     router=rng.choice([kind, kind, "f32"]))
            c["bias"] = c["scoring"] == "sigmoid" and rng.random() < 0.6
            cost = 3 * c["D"] * c["I"] * max(c["T"] * c["k"], 128 * E)
        if cost <= 8192 ** 3 // 2:
            return c


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(g, rows, cols, dtype):
    """Unit normal values with a few channels twenty times as large, as the
    inputs of transformer layers have them."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    big = torch.rand(cols, generator=g, device=DEV) < 0.003
    return torch.where(big, 20.0 * x, x).to(dtype)


def _stored4(g, rows, cols, low, high):
    """A 4-bit operand [rows, cols / 2] and its scales [rows, cols / 32], as checkpoints hold them: codes of
    normal values (a block's largest lies between 3.5 and 7), exponents between low and high."""
    pairs, blocks = -(-cols // 2), -(-cols // MX)
    v = torch.randn(rows, 2 * pairs, generator=g, device=DEV)
    m = v.abs()
    code = torch.zeros_like(v, dtype=torch.uint8)
    for border in (0.12, 0.36, 0.6, 0.84, 1.2, 1.7, 2.4):
        code += m > border
    code += 8 * (v < 0).to(torch.uint8)
    if cols % 2:
        code[:, -1] = 0
    q = code[:, 0::2] + 16 * code[:, 1::2]
    s = torch.randint(127 + low, 128 + high, (rows, blocks), generator=g, device=DEV, dtype=torch.int32)
    return q.view(torch.float4_e2m1fn_x2), s.to(torch.uint8).view(torch.float8_e8m0fnu)


def _weight8(g, *shape):
    """An 8-bit weight [..., N, K] and its scales [..., N / 128, K / 128], as
    checkpoints hold them."""
    N, K = shape[-2:]
    q = (torch.randn(*shape, generator=g, device=DEV) * 120.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = 1e-4 + 2e-4 * torch.rand(*shape[:-2], -(-N // BLOCK), -(-K // BLOCK), generator=g, device=DEV)
    return q, s


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["op"] == "quantize":
        s["x"] = _activations(g, case["M"], case["K"], TYPES[case["type"]])
    elif case["op"] == "mm":
        s["a"], s["a_scale"] = _stored4(g, case["M"], case["K"], -3, 2)
        s["b"], s["b_scale"] = _stored4(g, case["N"], case["K"], -8, -5)
    elif case["op"] == "linear":
        t = TYPES[case["type"]]
        s["x"] = _activations(g, case["M"], case["K"], t)
        s["w"], s["w_scale"] = _stored4(g, case["N"], case["K"], -8, -5)
        s["bias"] = (torch.randn(case["N"], generator=g, device=DEV) * 0.5).to(t) if case["bias"] else None
    elif case["op"] == "train":
        t = TYPES[case["type"]]
        s["x"] = _activations(g, case["M"], case["K"], t).requires_grad_()
        s["w"] = (0.02 * torch.randn(case["N"], case["K"], generator=g, device=DEV)).to(t).requires_grad_()
        s["dy"] = (0.01 * torch.randn(case["M"], case["N"], generator=g, device=DEV)).to(t)
    else:
        T, E, D, I = (case[n] for n in ("T", "E", "D", "I"))
        s["x"] = _activations(g, T, D, TYPES[case["type"]])
        # logits of about 1.5, some experts liked more than others
        r = torch.randn(E, D, generator=g, device=DEV) * (0.5 + torch.rand(E, 1, generator=g, device=DEV))
        s["router"] = (r * (1.2 / math.sqrt(D))).to(TYPES[case["router"]])
        s["bias"] = 0.1 * torch.randn(E, generator=g, device=DEV) if case["bias"] else None
        s["w1"], s["w1_scale"] = _weight8(g, E, 2, I, D)
        s["w2"], s["w2_scale"] = _weight8(g, E, D, I)
    return s


# The plain forms.


def _blocks4(x):
    """x's blocks of 32 along the last dimension: (values as e2m1 holds them, their power of two), in 32 bits."""
    x = x.float()
    b = torch.nn.functional.pad(x, (0, -x.shape[-1] % MX)).unflatten(-1, (-1, MX))
    m = b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    e = ((m.view(torch.int32) + 0x200000) >> 23) - 2  # m / 2^(e - 127) lies in [3.5, 7)
    s = (e << 23).view(torch.float32)
    v = b * torch.reciprocal(s)  # (a power of two: exact)
    a = v.abs()
    half, one, two = (torch.full_like(a, c) for c in (0.5, 1.0, 2.0))
    step = torch.where(a < 2.0, half, torch.where(a < 4.0, one, two))
    return torch.round(v / step) * step, s


def _rounded4(x, dim=-1):
    """x as its blocks of 32 along dim stand for it, in 32 bits."""
    q, s = _blocks4(x.movedim(dim, -1))
    return (q * s).flatten(-2)[..., :x.shape[dim]].movedim(-1, dim)


def _codes(q):
    """The values of a 4-bit operand, two a byte, in 32 bits."""
    u = q.view(torch.uint8)
    code = torch.stack((u & 15, u >> 4), -1).flatten(-2).int()
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
    return torch.where(code < 8, table[code & 7], -table[code & 7])


def _powers(s):
    return torch.exp2(s.view(torch.uint8).float() - 127.0)


def _values4(q, s):
    """A stored 4-bit operand [N, K / 2] with its scales, in 32 bits."""
    v = _codes(q)
    return v * _powers(s).repeat_interleave(MX, -1)[..., :v.shape[-1]]


def _plain_quantize(s):
    return _rounded4(s["x"]).to(s["x"].dtype)


def _plain_mm(s):
    c = _values4(s["a"], s["a_scale"]) @ _values4(s["b"], s["b_scale"]).t()
    return c.to(TYPES[s["case"]["out"]])


def _plain_linear(s):
    K = s["case"]["K"]
    y = _rounded4(s["x"]) @ _values4(s["w"], s["w_scale"])[:, :K].t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_train(s):
    x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
    y = _rounded4(x) @ _rounded4(w).t()
    dx = _rounded4(dy) @ _rounded4(w, 0)
    dw = _rounded4(dy, 0).t() @ _rounded4(x, 0)
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(w.dtype)}


def _route(c, x, bias):
    """(weights, ids) of FP32 logits x: the k experts of each token."""
    T, E, k, groups = c["T"], c["E"], c["k"], c["groups"]
    if c["scoring"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
        key = x
    else:
        p = torch.reciprocal(1.0 + torch.exp(-x))
        key = p if bias is None else p + bias
    if groups > 1:
        best = key.view(T, groups, -1).sort(dim=2, descending=True).values[:, :, :2]
        score = best.sum(2) if c["scoring"] == "sigmoid" else best[:, :, 0]
        kept = score.sort(dim=1, descending=True, stable=True).indices[:, :c["top"]]
        gone = torch.ones_like(score, dtype=torch.bool).scatter_(1, kept, False)
        key = key.masked_fill(gone.repeat_interleave(E // groups, 1), -math.inf)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :k]
    sel = p.gather(1, ids)
    return (sel / (sel.sum(1, keepdim=True) + 1e-20) if c["renormalize"] else sel), ids


def _rounded8(x):
    """x as its 8-bit blocks of 128 along the last dimension stand for it, in 32 bits."""
    K = x.shape[-1]
    b = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    m = b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    most = torch.full_like(m, 448.0)  # (tensors: torch divides by a number, or a number, through a reciprocal)
    q = (b * torch.div(most, m)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return (q * torch.div(m, most)).flatten(-2)[..., :K]


def _values8(q, s):
    """A stored 8-bit weight [..., N, K] with its scales, in 32 bits."""
    N, K = q.shape[-2:]
    s = s.repeat_interleave(BLOCK, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]
    return q.float() * s


def _plain_layer(s):
    c = s["case"]
    T, k, I = c["T"], c["k"], c["I"]
    # (in 64 bits: a choice between experts next to each other should not hang on the order of a sum)
    weights, ids = _route(c, (s["x"].double() @ s["router"].double().t()).float(), s["bias"])
    order = ids.flatten().sort(stable=True).indices  # slots by expert
    used, expert, count = torch.unique(ids.flatten()[order], return_inverse=True, return_counts=True)
    place = torch.arange(len(order), device=order.device) - (count.cumsum(0) - count)[expert]
    x = torch.zeros(len(used), int(count.max()), c["D"], device=order.device)
    x[expert, place] = _rounded8(s["x"])[order // k]
    w1, w2 = (_values8(s[n][used], s[n + "_scale"][used]) for n in ("w1", "w2"))  # of the experts in use
    gu = torch.bmm(x, w1.flatten(1, 2).transpose(1, 2).contiguous())
    gate, up = gu[:, :, :I], gu[:, :, I:]
    h = gate * torch.reciprocal(1.0 + torch.exp(-gate)) * up
    y = torch.bmm(_rounded8(h), w2.transpose(1, 2).contiguous())
    slots = torch.zeros(T * k, c["D"], device=order.device)
    slots[order] = y[expert, place] * weights.flatten()[order, None]
    return slots.view(T, k, -1).sum(1).to(s["x"].dtype)


def run(state):
    c = state["case"]
    if not own:
        return {"quantize": _plain_quantize, "mm": _plain_mm, "linear": _plain_linear, "train": _plain_train,
                "layer": _plain_layer}[c["op"]](state)
    from f16acc_amd import fp4, moe

    if c["op"] == "quantize":
        q, scale = fp4.quantize(state["x"])
        return fp4.dequantize(q, scale, state["x"].dtype)[:, :c["K"]]
    if c["op"] == "mm":
        return fp4.mm(state["a"], state["a_scale"], state["b"].t(), state["b_scale"].t(), TYPES[c["out"]])
    if c["op"] == "linear":
        return fp4.linear(state["x"], state["w"], state["w_scale"], state["bias"])
    if c["op"] == "train":
        y = fp4.linear(state["x"], state["w"])
        dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    return moe.layer(state["x"], state["router"], c["k"], state["w1"], state["w1_scale"], state["w2"],
                     state["w2_scale"], scoring=c["scoring"], bias=state["bias"], groups=c["groups"],
                     top_groups=c["top"], renormalize=c["renormalize"])


def work(case):
    def four(rows, cols):  # bytes of a 4-bit operand with its scales
        return rows * (-(-cols // 2) + -(-cols // MX))

    if case["op"] == "quantize":
        size = 4 if case["type"] == "f32" else 2
        n = case["M"] * case["K"]
        return {"bytes": 2 * size * n + four(case["M"], case["K"]), "flops": 4 * n}
    if case["op"] in ("mm", "linear", "train"):
        M, N, K = case["M"], case["N"], case["K"]
        size = 4 if case.get("type", case.get("out")) == "f32" else 2
        if case["op"] == "mm":
            return {"bytes": four(M, K) + four(N, K) + size * M * N, "flops": 2 * M * N * K}
        if case["op"] == "linear":
            return {"bytes": size * (M * K + M * N) + four(N, K) + (size * N if case["bias"] else 0),
                    "flops": 2 * M * N * K}
        return {"bytes": 2 * size * (M * K + N * K + M * N), "flops": 6 * M * N * K}
    T, E, k, D, I = (case[n] for n in ("T", "E", "k", "D", "I"))
    active = E * (1.0 - (1.0 - 1.0 / E) ** (T * k))  # experts that some token goes to
    router = E * D * (4 if case["router"] == "f32" else 2)
    return {"bytes": int(active * 3 * D * I + router + 4 * T * D), "flops": int(6 * T * k * D * I + 2 * T * E * D)}


# The definitions in 64 bits.


def _quantized4_64(x, dim=-1):
    """The 64-bit matrix x in blocks of 32 along dim, as they stand for it."""
    x = x.movedim(dim, -1)
    R, C = x.shape
    v = torch.zeros(R, -(-C // MX) * MX, dtype=torch.float64, device=x.device)
    v[:, :C] = x
    v = v.view(R, -1, MX)
    f, e = torch.frexp(v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100))  # f in [0.5, 1)
    s = torch.pow(torch.full_like(f, 2.0), (e - 3 + (f >= 0.875).int()).double())
    a, r = (v / s).abs(), torch.zeros_like(v)
    for i, (mid, step) in enumerate([(0.25, 0.5), (0.75, 0.5), (1.25, 0.5), (1.75, 0.5), (2.5, 1.0), (3.5, 1.0),
                                     (5.0, 2.0)]):
        r += step * ((a > mid) if i % 2 == 0 else (a >= mid))  # a tie goes to the even code
    r = (r * torch.sign(v) * s).view(R, -1)[:, :C]
    return r.movedim(-1, dim).contiguous()


def _stored4_64(q, s):
    u = q.view(torch.uint8).long()
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    both = torch.tensor(grid + [-v for v in grid], dtype=torch.float64, device=q.device)
    v = torch.empty(u.shape[0], 2 * u.shape[1], dtype=torch.float64, device=q.device)
    v[:, 0::2], v[:, 1::2] = both[u % 16], both[u // 16]
    block = torch.arange(v.shape[1], device=q.device) // MX
    e = s.view(torch.uint8).double() - 127.0
    return v * torch.pow(torch.full_like(e, 2.0), e)[:, block]


def _e4m3_64(v):
    """v rounded to the nearest e4m3 value, ties to even, in 64 bits."""
    v = v.clamp(-448.0, 448.0)
    _, e = torch.frexp(v)  # |v| in [2^(e-1), 2^e)
    step = torch.pow(torch.full_like(v, 2.0), (e - 4).clamp(min=-9).double())
    return torch.round(v / step) * step


def _quantized8_64(x):
    """The 64-bit matrix x in 8-bit blocks of 1 x 128, as they stand for it.  (Scale and reciprocal are FP32 by
    definition.)"""
    R, C = x.shape
    v = torch.zeros(R, -(-C // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :C] = x.float().double()
    v = v.view(R, -1, BLOCK)
    m = v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    scaled = (v * (448.0 / m).float().double()).float().double()
    return (_e4m3_64(scaled) * (m / 448.0).float().double()).view(R, -1)[:, :C].contiguous()


def _stored8_64(q, s):
    N, K = q.shape
    rows = torch.arange(N, device=q.device) // BLOCK
    cols = torch.arange(K, device=q.device) // BLOCK
    return q.double() * s.double()[rows][:, cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _quantized4_64(s["x"].double())
    if case["op"] == "mm":
        return _stored4_64(s["a"], s["a_scale"]) @ _stored4_64(s["b"], s["b_scale"]).t().contiguous()
    if case["op"] == "linear":
        w = _stored4_64(s["w"], s["w_scale"])[:, :case["K"]]
        y = _quantized4_64(s["x"].double()) @ w.t().contiguous()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "train":
        x, w, dy = (s[n].detach().double() for n in ("x", "w", "dy"))
        return {"y": _quantized4_64(x) @ _quantized4_64(w).t().contiguous(),
                "dx": _quantized4_64(dy) @ _quantized4_64(w, 0),
                "dw": _quantized4_64(dy, 0).t().contiguous() @ _quantized4_64(x, 0)}
    T, E, k, D = (case[n] for n in ("T", "E", "k", "D"))
    logits = (s["x"].double() @ s["router"].double().t().contiguous()).float()
    _, ids = _route(case, logits, s["bias"])  # (the choice is made on FP32 scores by definition)
    p = torch.sigmoid(logits.double()) if case["scoring"] == "sigmoid" else torch.softmax(logits.double(), 1)
    weights = p.gather(1, ids)
    if case["renormalize"]:
        weights = weights / (weights.sum(1, keepdim=True) + 1e-20)
    x = _quantized8_64(s["x"].double())
    y = torch.zeros(T, D, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if len(t) == 0:
            continue
        gate, up = (x[t] @ _stored8_64(s["w1"][e, i], s["w1_scale"][e, i]).t().contiguous() for i in (0, 1))
        h = _quantized8_64(gate * torch.sigmoid(gate) * up)
        out = h @ _stored8_64(s["w2"][e], s["w2_scale"][e]).t().contiguous()
        y.index_add_(0, t, out * weights[t, j][:, None])
    return y
