"""Plain 64-bit statements of the microscaled 4-bit operators, on the CPU, for the tests."""

import torch

F4, E8 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
MIDS = (GRID[1:] + GRID[:-1]) / 2
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def quantize(x):
    """(values [R, C] float64 as e2m1 holds them, exponents [R, blocks] int64, 128 for NaN) of a finite or
    non-finite x [R, C] in blocks of 1 x 32."""
    R, C = x.shape
    p = torch.zeros(R, -(-C // 32) * 32, dtype=torch.float64)
    p[:, :C] = x.detach().cpu().double()
    b = p.view(R, -1, 32)
    bad = ~torch.isfinite(b).all(-1)
    b = b.nan_to_num(0.0, 0.0, 0.0)
    m = b.abs().amax(-1).clamp(min=2.0 ** -100)
    _, e = torch.frexp(m / 3.5)  # m / 3.5 in [2^(e-1), 2^e)
    e = (e - 1).long()
    a = torch.ldexp(b.abs(), -e[..., None])
    q = torch.zeros_like(a)
    for i, mid in enumerate(MIDS):  # the step from code i to i + 1, taken at a tie if i is odd
        q += (GRID[i + 1] - GRID[i]) * ((a > mid) if i % 2 == 0 else (a >= mid))
    q = torch.copysign(q, b)
    return q.view(R, -1)[:, :C].clone(), torch.where(bad, 128, e)


def unpack(q, C=None):
    """The e2m1 values of q [R, P], float64."""
    u = q.detach().cpu().view(torch.uint8).long()
    both = torch.cat([GRID, -GRID])
    v = torch.stack((both[u % 16], both[u // 16]), -1).flatten(-2)
    return v if C is None else v[..., :C]


def scales(s):
    """2^e of e8m0 scales, NaN for 255, float64."""
    e = s.detach().cpu().view(torch.uint8).long()
    v = torch.ldexp(torch.ones(e.shape, dtype=torch.float64), e - 127)
    return torch.where(e == 255, torch.full_like(v, float("nan")), v)


def values(q, s, C=None):
    """What q [R, P] with scales s [R, blocks] stands for, its first C values, float64."""
    v = unpack(q)
    return (v * scales(s).repeat_interleave(32, -1)[..., :v.shape[-1]])[..., :C]


def rounded(x):
    """x [R, C] as its blocks stand for it."""
    q, e = quantize(x)
    s = torch.ldexp(torch.ones(e.shape, dtype=torch.float64), e)
    return q * torch.where(e == 128, torch.full_like(s, float("nan")), s).repeat_interleave(32, -1)[:, :x.shape[1]]


def check_product(c, a, b, bias=None):
    """c against a @ b.T (+ bias) in 64 bits, element by element.  A block's sum is exact.  A matrix instruction adds
    the sums of two blocks to an FP32 value: two additions off by 2^-23 (cut, not rounded) of at most the sum of all
    magnitudes each; the parts of a split, the bias and the result's rounding add as much a few times more."""
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        ref, mag = ref + bias.cpu().double(), mag + bias.cpu().double().abs()
    err = (c.detach().cpu().double() - ref).abs()
    adds = 2 * -(-a.shape[1] // 64) + 18
    bound = adds * 2.0 ** -23 * mag + ROUND[c.dtype] * ref.abs() + (2.0 ** -25 if c.dtype == torch.float16 else 0.0)
    assert torch.isfinite(c.detach()).all()
    assert bool((err <= bound).all()), f"off by {(err / bound.clamp(min=1e-300)).max().item():.2f} of the bound"
