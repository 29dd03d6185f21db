"""Plain 64-bit statements of the 8-bit block-scaled products and the
mixture-of-experts operators, on the CPU, for the tests."""

import torch

BLOCK = 128
MFMA = 1e-4  # bound of an fp8 MFMA's sum of 128 products, relative to the sum of their magnitudes (measured: 5e-5)
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -22}


def e4m3(v):
    """Nearest e4m3 value, ties to even, by arithmetic."""
    v = v.clamp(-448.0, 448.0)
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return torch.round(v / step) * step


def quantize(x, rows=1, cols=BLOCK):
    """(values [R, C] float64, scales [R / rows, C / cols] float32) of x [R, C] in blocks of rows x cols."""
    R, C = x.shape
    p = torch.zeros(-(-R // rows) * rows, -(-C // cols) * cols, dtype=torch.float64)
    p[:R, :C] = x.detach().cpu().float().double()
    b = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    m = b.abs().amax(dim=(1, 3), keepdim=True).clamp(min=2.0 ** -100)
    q = e4m3((b * (448.0 / m).float().double()).float().double())
    return q.view_as(p)[:R, :C].clone(), (m / 448.0).float().view(p.shape[0] // rows, -1)


def values(q, s, rows=1, cols=BLOCK):
    """What q [R, C] with scales s [R / rows, C / cols] stands for, float64."""
    R, C = q.shape
    s = s.detach().cpu().double().repeat_interleave(rows, 0)[:R].repeat_interleave(cols, 1)[:, :C]
    return q.detach().cpu().float().double() * s


def rounded(x, rows=1, cols=BLOCK):
    return values(*quantize(x, rows, cols), rows, cols)


def check_product(c, a, b, bias=None):
    """c against a @ b.T (+ bias) in 64 bits, element by element: the MFMA's bound on the sum, one rounding."""
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        ref, mag = ref + bias.cpu().double(), mag + bias.cpu().double().abs()
    err = (c.detach().cpu().double() - ref).abs()
    bound = MFMA * mag + ROUND[c.dtype] * ref.abs() + (2.0 ** -24 if c.dtype == torch.float16 else 0.0)
    assert torch.isfinite(c.detach()).all()
    assert bool((err <= bound).all()), f"off by {(err / bound.clamp(min=1e-300)).max().item():.2f} of the bound"


def route(logits, k, scoring="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    """(weights float64, ids int64, smallest distance of a chosen key to one left out or chosen after it), token by token."""
    x = logits.detach().cpu().double()
    T, E = x.shape
    out_w, out_i = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1)
    p_all, gap = torch.zeros(T, E, dtype=torch.float64), float("inf")
    for t in range(T):
        row = x[t]
        if scoring == "softmax":
            p = torch.softmax(row, 0) if bool((row > -float("inf")).any()) else torch.zeros(E, dtype=torch.float64)
        else:
            p = torch.sigmoid(row)
        p_all[t] = p
        key = row.clone() if scoring == "softmax" and bias is None else p + (0 if bias is None else bias.cpu().double())
        key[(row == -float("inf")) | torch.isnan(row)] = -float("inf")
        if groups > 1:
            per = key.view(groups, -1)
            if scoring == "softmax":
                score = per.amax(1)
            else:
                best = per.sort(dim=1, descending=True).values[:, :2]
                score = best[:, 0] + (best[:, 1].masked_fill(best[:, 1] == -float("inf"), 0) if best.shape[1] > 1 else 0)
            kept = sorted(range(groups), key=lambda g: (-score[g].item(), g))[:top_groups]
            for g in range(groups):
                if g not in kept:
                    per[g] = -float("inf")
        order = sorted((e for e in range(E) if key[e] > -float("inf")), key=lambda e: (-key[e].item(), e))
        for a, b in zip(order[:k], order[1:k + 1]):
            d = key[a].item() - key[b].item()
            gap = min(gap, d if d > 0 else gap)
        chosen = order[:k]
        w = p[chosen]
        if renormalize:
            w = w / (w.sum() + 1e-20)
        out_w[t, :len(chosen)] = w * scale
        out_i[t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int64)
    return out_w, out_i, gap


def route_grad(logits, ids, dw, scoring="softmax", renormalize=True, scale=1.0):
    x = logits.detach().cpu().double().requires_grad_()
    if scoring == "softmax":  # (a row without an available expert has p = 0 and no gradient)
        live = (x.detach() > -float("inf")).any(1, keepdim=True)
        p = torch.softmax(torch.where(live, x, torch.zeros_like(x)), 1) * live
    else:
        p = torch.sigmoid(x)
    sel = torch.where(ids >= 0, p.gather(1, ids.clamp(min=0)), 0.0)
    w = scale * (sel / (sel.sum(1, keepdim=True) + 1e-20) if renormalize else sel)
    return torch.autograd.grad(w, x, dw.cpu().double())[0]


def experts(x, weights, ids, w1, s1, w2, s2):
    """The routed experts' FFN in 64 bits, the hidden values quantised from 64 bits."""
    xq = rounded(x)
    y = torch.zeros(x.shape, dtype=torch.float64)
    for e in range(w1.shape[0]):
        t, j = (ids.cpu() == e).nonzero(as_tuple=True)
        if len(t) == 0:
            continue
        gate, up = (xq[t] @ values(w1[e, i], s1[e, i], BLOCK).t() for i in (0, 1))
        h = rounded_64(gate * torch.sigmoid(gate) * up)
        y.index_add_(0, t, h @ values(w2[e], s2[e], BLOCK).t() * weights.cpu().double()[t, j][:, None])
    return y


def rounded_64(h):
    return rounded(h.float())
