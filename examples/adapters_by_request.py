"""Many adapters beside one projection: a batch is served, then the adapters are trained.

A w8 projection [768, 512] is shared by four adapters. A batch of requests of ragged lengths, each with its adapter,
runs in one call; then every adapter learns a target change of the weight from its own requests' rows: the forward pass
keeps its input in 8 bits and the rank-space rows in f32, the backward pass reads both, and Adam on f32 master copies
writes the factors back into the bank.

    python examples/adapters_by_request.py [steps]
"""
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "vpipe-ming-image_b200"))

from mingproj import pack as P  # noqa: E402
from mingproj.proj import Context  # noqa: E402


def main(steps: int = 40, seed: int = 0) -> list[float]:
    n, k, adapters, rank = 768, 512, 4, 16
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    ctx = Context(torch.cuda.current_device())
    packed = P.synthetic_affine(rng, n, k, 8)
    w = ctx.upload(n, k, 8, packed.data, packed.scales, packed.biases)
    wt = ctx.transposed(w)  # for the gradient of x

    # master copies in f32, the bank's in bf16; B starts at zero: an adapter that has not learnt adds nothing
    a = normal(adapters, rank, k, std=k ** -0.5)
    b = torch.zeros(adapters, n, rank, device="cuda")
    bank = ctx.adapters(n, k, adapters, rank, training=True)

    def load():
        for i in range(adapters):
            bank.set(i, a[i].bfloat16(), b[i].bfloat16())

    load()
    # the change each adapter is to learn: of rank 4
    goal = normal(adapters, n, 4, std=0.5) @ normal(adapters, 4, k, std=k ** -0.5)

    lengths, owner = [97, 300, 1, 128, 0, 250, 64], [0, 1, 2, 3, 0, 2, -1]  # -1: a request without an adapter
    m = sum(lengths)
    plan = ctx.requests(len(lengths), m, adapters)
    plan.plan(lengths, owner)
    rows = torch.tensor(np.repeat(owner, lengths), device="cuda")

    # one new token of each request that has an adapter, as a serving loop would ask for them
    few = ctx.requests(4, 4, adapters)
    few.plan([1, 1, 1, 1], [0, 1, 2, 3])
    token = normal(4, k).bfloat16()
    before = ctx.linear_requests(w, token, bank, few)

    first, second = [torch.zeros_like(a), torch.zeros_like(b)], [torch.zeros_like(a), torch.zeros_like(b)]
    losses = []
    for step in range(1, steps + 1):
        x = normal(m, k).bfloat16()
        y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
        saved = ctx.checkpoint(x)
        target = ctx.linear(w, x).float()
        for i in range(adapters):
            target[rows == i] += x[rows == i].float() @ goal[i].T
        off = y.float() - target
        losses.append(float(off.square().sum(1).mean()))
        dx, da, db = ctx.linear_requests_grad(wt, (2.0 * off).bfloat16(), saved, v, bank, plan)
        count = torch.tensor([max(1, int((rows == i).sum())) for i in range(adapters)], device="cuda")[:, None, None]
        for i, grad in enumerate((da / count, db / count)):
            first[i].mul_(0.9).add_(grad, alpha=0.1)
            second[i].mul_(0.99).addcmul_(grad, grad, value=0.01)
            size = (second[i] / (1 - 0.99 ** step)).sqrt() + 1e-8
            (a, b)[i].addcdiv_(first[i], size, value=-0.02 / (1 - 0.9 ** step))
        load()
    after = ctx.linear_requests(w, token, bank, few)
    ctx.sync_check()
    change = (after - before).float().norm() / before.float().norm()
    print(f"loss a row: {losses[0]:.3f} -> {losses[-1]:.3f} in {steps} steps; a new token's output moved by {change:.2f}")
    for h in (few, plan, bank, wt, w):
        h.free()
    ctx.close()
    return losses


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 40)
