"""A transformer's mixture-of-experts block in 8 bits: quantise, serve, train.

    python examples/moe_block.py

1. A block's 16-bit weights are quantised once (fp8.quantize_weight).
2. A prompt and then single tokens go through it: an FP16 router layer on the
   chunked GEMM (f16acc_amd.enable), moe.route, moe.experts, and a shared dense
   layer on fp8.linear.  A token must come out the same alone as in its prompt, up to the
   rounding of the kernels for few and for many tokens.
3. The dense layer is trained against a teacher with both directions in 8 bits
   (fp8.linear on a 16-bit weight), and the router through the gradient of
   moe.route.
"""

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import f16acc_amd as f16acc  # noqa: E402
from f16acc_amd import fp8, moe  # noqa: E402


class MoeBlock:
    """E experts of a gated feed-forward D -> I -> D, k of them a token, beside a dense layer."""

    def __init__(self, D, I, E, k, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape, fan):
            return torch.randn(*shape, generator=g, device=device).mul_(fan ** -0.5).half()

        self.k = k
        self.router = weight(E, D, fan=D)
        self.w1 = fp8.quantize_weight(weight(E, 2, I, D, fan=D))
        self.w2 = fp8.quantize_weight(weight(E, D, I, fan=I))
        self.shared = fp8.quantize_weight(weight(D, D, fan=D))

    @torch.inference_mode()
    def __call__(self, x):
        logits = F.linear(x, self.router)
        weights, ids = moe.route(logits, self.k)
        return moe.experts(x, weights, ids, *self.w1, *self.w2) + fp8.linear(x, *self.shared)


def serve(block, x):
    """The prompt at once, then its first tokens one by one: the largest relative distance of a token's results."""
    prompt = block(x)
    far = 0.0
    for t in range(8):
        alone = block(x[t:t + 1])[0].float()
        far = max(far, ((alone - prompt[t].float()).norm() / prompt[t].float().norm()).item())
    return far


def train(x, D, E, k, steps=40, device="cuda"):
    """Adam on a dense layer and a router towards a teacher's: (first, last) loss of each."""
    g = torch.Generator(device=device).manual_seed(1)
    teacher = torch.randn(D, D, generator=g, device=device).mul_(D ** -0.5).to(x.dtype)
    wanted = moe.route(x @ torch.randn(D, E, generator=g, device=device).mul_(D ** -0.5).to(x.dtype), k)
    w = torch.zeros(D, D, dtype=x.dtype, device=device, requires_grad=True)
    router = torch.randn(E, D, generator=g, device=device).mul_(D ** -0.5).requires_grad_()
    opt = torch.optim.Adam([w, router], lr=2e-3)
    target, losses = x @ teacher, []
    for _ in range(steps):
        dense = (fp8.linear(x, w).float() - target.float()).square().mean()
        weights, ids = moe.route(x.float() @ router.t(), E)  # every expert's weight, to compare with the wanted ones
        mine = torch.zeros_like(weights).scatter(1, ids.long(), weights)
        want = torch.zeros_like(weights).scatter(1, wanted[1].long(), wanted[0])
        routing = -(want * (mine + 1e-9).log()).sum(1).mean()
        opt.zero_grad()
        (dense + routing).backward()
        opt.step()
        losses.append((dense.item(), routing.item()))
    return tuple(zip(losses[0], losses[-1]))


def main(tokens=512, D=1024, I=512, E=32, k=4):
    f16acc.enable()
    try:
        g = torch.Generator(device="cuda").manual_seed(2)
        x = torch.randn(tokens, D, generator=g, device="cuda").half()
        far = serve(MoeBlock(D, I, E, k), x)
        print(f"{tokens} tokens, {E} experts, {k} each: a token alone is within {far:.1e} of itself in the prompt")
        dense, routing = train(x.bfloat16(), D, E, k)
        print(f"dense layer in 8 bits: loss {dense[0]:.3f} -> {dense[1]:.3f};  router: {routing[0]:.3f} -> {routing[1]:.3f}")
        return far, dense, routing
    finally:
        f16acc.disable()


if __name__ == "__main__":
    main()
