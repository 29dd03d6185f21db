"""Cases of the 8-bit block-scaled products and of the mixture-of-experts
operators: f16acc_amd.fp8 and f16acc_amd.moe.

"linear"   fp8.linear(x, w, w_scale, bias): 16-bit activations quantised in
           blocks of 1 x 128, times a stored 8-bit weight with a scale for each
           128 x 128 block.
"train"    the same layer on a 16-bit weight, forward and backward: y, dx, dw.
"route"    moe.route: expert scores to the k experts of each token and their
           weights, with the gradient of the scores where a case trains.
"experts"  moe.experts: the routed tokens through their experts' gated FFN in
           8 bits (gate and up, SiLU, down, weighted sum).

A block of x is quantised as s = m / 448 with m = max(|x|, 2^-100), and
q = e4m3(x * (448 / m)), each step rounded once to FP32.
"""

import math

import torch

# False: run() computes the plain forms below.  True: it calls the framework.
own = False

DEV = "cuda"
BLOCK = 128
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One token through the widest layer of Qwen2.5-1.5B (gate/up): a decode
        # step, whose cost is reading the weight and the call itself.
        dict(name="linear_token", op="linear", M=1, N=8960, K=1536, type="f16", bias=False),
        # A short batch against a weight whose rows no 16-byte load fits.
        dict(name="linear_odd_77", op="linear", M=77, N=1537, K=8961, type="bf16", bias=True),
        # The same gate/up layer over a prompt of 2048 tokens.
        dict(name="linear_gateup_2048", op="linear", M=2048, N=8960, K=1536, type="f16", bias=True),
        # The largest product: the square the 16-bit GEMM is measured on.
        dict(name="linear_8192", op="linear", M=8192, N=8192, K=8192, type="bf16", bias=False),
        # Training steps of the q/o projection and of the down projection.
        dict(name="train_qo_2048", op="train", M=2048, N=1536, K=1536, type="bf16"),
        dict(name="train_down_4096", op="train", M=4096, N=1536, K=8960, type="f16"),
        # Routing of a decode batch of eight sequences.
        dict(name="route_8", op="route", T=8, E=64, k=6, type="f32", scoring="softmax", bias=False, groups=1, top=1,
             renormalize=True, masked=0.0, grad=False),
        # A training batch of odd size: 16-bit scores, experts masked out, a
        # few padding tokens with every expert masked.
        dict(name="route_odd_1001", op="route", T=1001, E=60, k=4, type="bf16", scoring="softmax", bias=False,
             groups=1, top=1, renormalize=False, masked=0.1, grad=True),
        # The widest: sigmoid scores with a balance bias, 8 groups of 32
        # experts of which 4 stay, a training batch of 16384 tokens.
        dict(name="route_16384", op="route", T=16384, E=256, k=8, type="f32", scoring="sigmoid", bias=True, groups=8,
             top=4, renormalize=True, masked=0.0, grad=True),
        # One token through six of 64 experts: reading their weights.
        dict(name="experts_token", op="experts", T=1, E=64, k=6, D=2048, I=1024, type="f16", dropped=0.0),
        # A ragged batch: widths that end inside a block, tokens without experts.
        dict(name="experts_odd_77", op="experts", T=77, E=20, k=3, D=1040, I=720, type="bf16", dropped=0.1),
        # A prompt of 4096 tokens over 64 experts.
        dict(name="experts_4096", op="experts", T=4096, E=64, k=8, D=2048, I=1024, type="bf16", dropped=0.0),
    ]


def _extent(rng, lo, hi, odd=0.15):
    """An extent spread over its logarithm: mostly multiples of 128, else of
    16, else any number."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    r = rng.random()
    step = 1 if r < odd else 16 if r < 0.4 else 128
    return max(lo, min(hi, v // step * step))


def draw(rng):
    op = rng.choice(["linear", "linear", "train", "route", "experts", "experts"])
    kind = rng.choice(["f16", "bf16"])
    while True:
        if op == "linear":
            c = dict(op=op, M=_extent(rng, 1, 8192, odd=0.6), N=_extent(rng, 128, 16384), K=_extent(rng, 128, 12288),
                     type=kind, bias=rng.random() < 0.5)
            cost = c["M"] * c["N"] * c["K"]
        elif op == "train":
            c = dict(op=op, M=_extent(rng, 128, 8192), N=_extent(rng, 128, 8960), K=_extent(rng, 128, 8960), type=kind)
            cost = 3 * c["M"] * c["N"] * c["K"]
        elif op == "route":
            groups = rng.choice([1, 1, 4, 8])
            E = groups * rng.randint(max(1, 8 // groups), 256 // groups)
            top = rng.randint(1, groups)
            c = dict(op=op, T=_extent(rng, 1, 16384, odd=0.6), E=E, k=rng.randint(1, min(8, top * E // groups)),
                     type=rng.choice(["f16", "bf16", "f32"]), scoring=rng.choice(["softmax", "sigmoid"]), bias=False,
                     groups=groups, top=top, renormalize=rng.random() < 0.7, masked=rng.choice([0.0, 0.0, 0.1]),
                     grad=rng.random() < 0.6)
            c["bias"] = c["scoring"] == "sigmoid" and rng.random() < 0.6
            if c["k"] == 1:
                c["renormalize"] = False  # (one weight, always 1, has no gradient)
            if c["T"] < 16:
                c["masked"] = 0.0
            cost = 0
        else:
            E = rng.randint(8, 128)
            c = dict(op=op, T=_extent(rng, 1, 8192, odd=0.6), E=E, k=rng.randint(1, 8),
                     D=_extent(rng, 256, 4096, odd=0.0), I=_extent(rng, 256, 2048, odd=0.0), type=kind,
                     dropped=rng.choice([0.0, 0.0, 0.1]))
            if c["T"] < 16:
                c["dropped"] = 0.0
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


def _weight(g, *shape):
    """An 8-bit weight [..., N, K] and its scales [..., N / 128, K / 128], as
    checkpoints hold them."""
    N, K = shape[-2:]
    q = (torch.randn(*shape, generator=g, device=DEV) * 120.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = 1e-4 + 2e-4 * torch.rand(*shape[:-2], -(-N // BLOCK), -(-K // BLOCK), generator=g, device=DEV)
    return q, s


def prepare(case, seed):
    g = _generator(seed)
    t = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "linear":
        s["x"] = _activations(g, case["M"], case["K"], t)
        s["w"], s["w_scale"] = _weight(g, case["N"], case["K"])
        s["bias"] = (torch.randn(case["N"], generator=g, device=DEV) * 0.5).to(t) if case["bias"] else None
    elif case["op"] == "train":
        s["x"] = _activations(g, case["M"], case["K"], t).requires_grad_()
        s["w"] = (0.02 * torch.randn(case["N"], case["K"], generator=g, device=DEV)).to(t).requires_grad_()
        s["dy"] = (0.01 * torch.randn(case["M"], case["N"], generator=g, device=DEV)).to(t)
    elif case["op"] == "route":
        T, E = case["T"], case["E"]
        # tokens' scores, some experts liked more than others
        x = 1.5 * torch.randn(T, E, generator=g, device=DEV) + 0.5 * torch.randn(E, generator=g, device=DEV)
        if case["masked"]:
            x.masked_fill_(torch.rand(T, E, generator=g, device=DEV) < case["masked"], -math.inf)
            x.masked_fill_(torch.rand(T, 1, generator=g, device=DEV) < 0.02, -math.inf)
        s["logits"] = x.to(t).requires_grad_(case["grad"])
        s["bias"] = 0.1 * torch.randn(E, generator=g, device=DEV) if case["bias"] else None
        s["dw"] = torch.randn(T, case["k"], generator=g, device=DEV)
    else:
        T, E, k, D, I = (case[n] for n in ("T", "E", "k", "D", "I"))
        s["x"] = _activations(g, T, D, t)
        score = torch.randn(T, E, generator=g, device=DEV) + 0.5 * torch.randn(E, generator=g, device=DEV)
        top, ids = score.topk(k, dim=1)
        s["weights"] = torch.softmax(top, dim=1)
        gone = torch.rand(T, k, generator=g, device=DEV) < case["dropped"]
        s["ids"] = ids.to(torch.int32).masked_fill_(gone, -1)
        s["w1"], s["w1_scale"] = _weight(g, E, 2, I, D)
        s["w2"], s["w2_scale"] = _weight(g, E, D, I)
    return s


# The plain forms.


def _blocks(x, dim):
    """x in 32 bits and in blocks of 128 along dim (the last or the one before
    it), quantised: (values as e4m3 holds them, scales, one a block)."""
    x = x.float().movedim(dim, -1)
    K = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    m = b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    most = torch.full_like(m, 448.0)  # (tensors: torch divides by a number, or a number, through a reciprocal)
    q = (b * torch.div(most, m)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return q, torch.div(m, most)


def _rounded(x, dim=-1):
    """x as its blocks of 128 along dim stand for it, in 32 bits."""
    q, s = _blocks(x, dim)
    return (q * s).flatten(-2)[..., :x.shape[dim]].movedim(-1, dim)


def _rounded_weight(w):
    """A [N, K] weight as its 128 x 128 blocks stand for it, in 32 bits."""
    N, K = w.shape
    b = torch.nn.functional.pad(w.float(), (0, -K % BLOCK, 0, -N % BLOCK))
    b = b.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK))  # [N / 128, 128, K / 128, 128]
    m = b.abs().amax((1, 3), keepdim=True).clamp(min=2.0 ** -100)
    most = torch.full_like(m, 448.0)
    q = (b * torch.div(most, m)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return (q * torch.div(m, most)).flatten(2).flatten(0, 1)[:N, :K]


def _values(q, s):
    """A stored weight [..., N, K] with its scales, in 32 bits."""
    N, K = q.shape[-2:]
    s = s.repeat_interleave(BLOCK, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]
    return q.float() * s


def _plain_linear(s):
    y = _rounded(s["x"]) @ _values(s["w"], s["w_scale"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_train(s):
    x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
    wq = _rounded_weight(w)
    y = _rounded(x) @ wq.t()
    dx = _rounded(dy) @ wq
    dw = _rounded(dy, 0).t() @ _rounded(x, 0)
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(w.dtype)}


def _plain_route(s):
    c = s["case"]
    T, E, k, groups = c["T"], c["E"], c["k"], c["groups"]
    x = s["logits"].detach().float()
    if c["scoring"] == "softmax":
        m = x.amax(1, keepdim=True)
        e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
        total = e.sum(1, keepdim=True)
        p = torch.where(total > 0, e / total, e)
        key = x
    else:
        p = torch.reciprocal(1.0 + torch.exp(-x))
        key = p if s["bias"] is None else p + s["bias"]
        key = key.masked_fill(x == -math.inf, -math.inf)
    if groups > 1:
        best = key.view(T, groups, -1).sort(dim=2, descending=True).values[:, :, :2]
        score = best[:, :, 0]
        if c["scoring"] == "sigmoid" and best.shape[2] > 1:
            score = score + best[:, :, 1].masked_fill(best[:, :, 1] == -math.inf, 0.0)
        kept = score.sort(dim=1, descending=True, stable=True).indices[:, :c["top"]]
        gone = torch.ones_like(score, dtype=torch.bool).scatter_(1, kept, False)
        key = key.masked_fill(gone.repeat_interleave(E // groups, 1), -math.inf)
    top, ids = (v[:, :k] for v in key.sort(dim=1, descending=True, stable=True))
    none = top == -math.inf
    sel = p.gather(1, ids).masked_fill(none, 0.0)
    total = sel.sum(1, keepdim=True) + 1e-20
    weights = sel / total if c["renormalize"] else sel
    out = {"weights": weights, "ids": ids.to(torch.int32).masked_fill(none, -1)}
    if c["grad"]:
        dp = s["dw"]
        if c["renormalize"]:
            dp = dp / total - (dp * sel).sum(1, keepdim=True) / (total * total)
        dp = torch.zeros_like(p).scatter_(1, ids, dp.masked_fill(none, 0.0))
        if c["scoring"] == "softmax":
            dx = p * (dp - (dp * p).sum(1, keepdim=True))
        else:
            dx = dp * p * (1.0 - p)
        out["dlogits"] = dx.to(s["logits"].dtype)
    return out


def _plain_experts(s):
    c = s["case"]
    T, k, I = c["T"], c["k"], c["I"]
    ids = s["ids"].long().flatten()
    order = ids.sort(stable=True).indices  # slots by expert, those without one first
    order = order[(ids == -1).sum():]
    used, expert, count = torch.unique(ids[order], return_inverse=True, return_counts=True)
    place = torch.arange(len(order), device=order.device) - (count.cumsum(0) - count)[expert]
    x = torch.zeros(len(used), int(count.max()), c["D"], device=order.device)
    x[expert, place] = _rounded(s["x"])[order // k]
    w1, w2 = (_values(s[n][used], s[n + "_scale"][used]) for n in ("w1", "w2"))  # of the experts in use
    gu = torch.bmm(x, w1.flatten(1, 2).transpose(1, 2).contiguous())
    gate, up = gu[:, :, :I], gu[:, :, I:]
    h = gate * torch.reciprocal(1.0 + torch.exp(-gate)) * up
    y = torch.bmm(_rounded(h), w2.transpose(1, 2).contiguous())
    slots = torch.zeros(T * k, c["D"], device=order.device)
    slots[order] = y[expert, place] * s["weights"].flatten()[order, None]
    return slots.view(T, k, -1).sum(1).to(s["x"].dtype)


def run(state):
    c = state["case"]
    if not own:
        return {"linear": _plain_linear, "train": _plain_train, "route": _plain_route,
                "experts": _plain_experts}[c["op"]](state)
    from f16acc_amd import fp8, moe

    if c["op"] == "linear":
        return fp8.linear(state["x"], state["w"], state["w_scale"], state["bias"])
    if c["op"] == "train":
        y = fp8.linear(state["x"], state["w"])
        dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if c["op"] == "route":
        weights, ids = moe.route(state["logits"], c["k"], scoring=c["scoring"], bias=state["bias"],
                                 groups=c["groups"], top_groups=c["top"], renormalize=c["renormalize"])
        out = {"weights": weights, "ids": ids}
        if c["grad"]:
            out["dlogits"], = torch.autograd.grad(weights, state["logits"], state["dw"])
        return out
    return moe.experts(state["x"], state["weights"], state["ids"], state["w1"], state["w1_scale"], state["w2"],
                       state["w2_scale"])


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        scales = 4 * -(-N // BLOCK) * -(-K // BLOCK)
        return {"bytes": size * (M * K + M * N) + N * K + scales + (size * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    if case["op"] == "train":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * size * (M * K + N * K + M * N), "flops": 6 * M * N * K}
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        n = size * T * E + 8 * T * k + (4 * E if case["bias"] else 0)
        return {"bytes": n + (size * T * E + 4 * T * k if case["grad"] else 0), "flops": 10 * T * E}
    T, E, k, D, I = (case[n] for n in ("T", "E", "k", "D", "I"))
    slots = T * k * (1.0 - case["dropped"])
    active = E * (1.0 - (1.0 - 1.0 / E) ** slots)  # experts that some token goes to
    return {"bytes": int(active * 3 * D * I + 2 * size * T * D + 8 * T * k), "flops": int(6 * slots * D * I)}


# The definitions in 64 bits.


def _e4m3_64(v):
    """v rounded to the nearest e4m3 value, ties to even, in 64 bits."""
    v = v.clamp(-448.0, 448.0)
    _, e = torch.frexp(v)  # |v| in [2^(e-1), 2^e)
    step = torch.pow(torch.full_like(v, 2.0), (e - 4).clamp(min=-9).double())
    return torch.round(v / step) * step


def _quantized_64(x, rows, cols):
    """The 64-bit matrix x in blocks of rows x cols, as their e4m3 values and
    FP32 scales stand for it.  (Scale and reciprocal are FP32 by definition.)"""
    R, C = x.shape
    out = torch.zeros(-(-R // rows) * rows, -(-C // cols) * cols, dtype=torch.float64, device=x.device)
    out[:R, :C] = x.float().double()
    v = out.view(-1, rows, out.shape[1] // cols, cols)
    m = v.abs().amax(dim=(1, 3), keepdim=True).clamp(min=2.0 ** -100)
    scaled = (v * (448.0 / m).float().double()).float().double()
    return (_e4m3_64(scaled) * (m / 448.0).float().double()).view_as(out)[:R, :C].contiguous()


def _stored_64(q, s):
    N, K = q.shape
    rows = torch.arange(N, device=q.device) // BLOCK
    cols = torch.arange(K, device=q.device) // BLOCK
    return q.double() * s.double()[rows][:, cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = _quantized_64(s["x"].double(), 1, BLOCK) @ _stored_64(s["w"], s["w_scale"]).t().contiguous()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "train":
        x, w, dy = (s[n].detach().double() for n in ("x", "w", "dy"))
        qw = _quantized_64(w, BLOCK, BLOCK)
        y = _quantized_64(x, 1, BLOCK) @ qw.t().contiguous()
        dx = _quantized_64(dy, 1, BLOCK) @ qw
        dw = _quantized_64(dy, BLOCK, 1).t().contiguous() @ _quantized_64(x, BLOCK, 1)
        return {"y": y, "dx": dx, "dw": dw}
    if case["op"] == "route":
        x = s["logits"].detach().double()
        p = torch.sigmoid(x) if case["scoring"] == "sigmoid" else torch.softmax(x, 1).nan_to_num(0.0)
        p.requires_grad_()
        ids = _plain_route(s)["ids"].long()  # (whole numbers: the choice itself is compared apart)
        sel = torch.where(ids >= 0, p.gather(1, ids.clamp(min=0)), 0.0)
        w = sel / (sel.sum(1, keepdim=True) + 1e-20) if case["renormalize"] else sel
        out = {"weights": w.detach(), "ids": None}
        if case["grad"]:
            dp, = torch.autograd.grad(w, p, s["dw"].double())
            p = p.detach()
            out["dlogits"] = (dp * p * (1.0 - p) if case["scoring"] == "sigmoid"
                              else p * (dp - (dp * p).sum(1, keepdim=True)))
        return out
    T, E, k, D = case["T"], case["E"], case["k"], case["D"]
    x = _quantized_64(s["x"].double(), 1, BLOCK)
    y = torch.zeros(T, D, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, j = (s["ids"] == e).nonzero(as_tuple=True)
        if len(t) == 0:
            continue
        gate, up = (x[t] @ _stored_64(s["w1"][e, i], s["w1_scale"][e, i]).t().contiguous() for i in (0, 1))
        h = _quantized_64(gate * torch.sigmoid(gate) * up, 1, BLOCK)
        out = h @ _stored_64(s["w2"][e], s["w2_scale"][e]).t().contiguous()
        y.index_add_(0, t, out * s["weights"].double()[t, j][:, None])
    return y
